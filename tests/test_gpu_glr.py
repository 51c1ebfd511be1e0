"""The gated linear recurrence on the GPU against its definition in 64 bits: sizes, types, layouts, masks, edges, streams and
graphs.  Tolerances are the worst cases derived in tests/glr_reference.py plus half a step of the output's type."""
import pytest
import torch

from tests import glr_reference as ref

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def hip():
    from baselines_amd import hip
    return hip


def half_step(t):
    return torch.finfo(t).eps / 2


def layout(kind, T, E, H, dtype, fill):
    """[T, E, H] tensor of the given layout with values from `fill`, and the buffer that it lives in."""
    if kind == "joint":
        buf = torch.empty((T, E, 2 * H), dtype=dtype, device="cuda")
        t = buf[..., H:]
    elif kind == "batch first":
        buf = torch.empty((E, T, H), dtype=dtype, device="cuda")
        t = buf.transpose(0, 1)
    elif kind == "odd":                     # rows at odd addresses, gaps between rows and steps
        buf = torch.empty(3 + T * (E * (H + 3) + 5), dtype=dtype, device="cuda")
        t = buf[3:].as_strided((T, E, H), (E * (H + 3) + 5, H + 3, 1), 3)
    else:
        buf = t = torch.empty((T, E, H), dtype=dtype, device="cuda")
    if fill is not None:
        t.copy_(fill)
    return t, buf


def make(T, E, H, dtype, kind="apart", resets=False, bias=False, h0=True, seed=0, reach=6.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *s: torch.randn(s, generator=g, device="cuda")      # noqa: E731
    f = layout(kind, T, E, H, dtype, normal(T, E, H) + (0 if bias else 1) * reach * torch.rand(H, generator=g, device="cuda"))[0]
    x = layout(kind, T, E, H, dtype, normal(T, E, H))[0]
    return dict(f=f, x=x, h0=normal(E, H) if h0 else None,
                resets=(torch.rand((T, E), generator=g, device="cuda") < 0.1) if resets else None,
                bias=reach * torch.rand(H, generator=g, device="cuda") if bias else None), normal


def close(got, want, tol, what):
    """|got - want| <= tol + half a step of got's type at the value."""
    assert got.shape == want.shape, what
    err = (got.double() - want).abs()
    bound = tol + (half_step(got.dtype) * want.abs() if got.dtype != torch.float32 else 0.0)
    if got.dtype == F16:
        bound = bound + 2.0 ** -25          # half a step of the smallest float16 numbers
    if got.dtype != torch.float32:
        bound = bound * (1 + 2 * half_step(got.dtype))
    bad = ~(err <= bound)
    assert not bool(bad.any()), (what, float(err[bad].max()), "of bound", float((err / bound.clamp(min=1e-300)).max()), int(bad.sum()))


def check(hip, a, normal, dtype, kind="apart", dh_last=True, backward=True):
    T, E, H = a["x"].shape
    y, h_last, saved = hip.glr_forward(a["f"], a["x"], a["h0"], resets=a["resets"], bias=a["bias"], want_saved=True)
    want, last, _ = ref.forward(a["f"], a["x"], a["h0"], a["resets"], a["bias"])
    b = ref.Bounds(a["f"], a["x"], a["h0"], a["resets"], a["bias"])
    assert y.dtype == dtype and h_last.dtype == F32
    close(y, want, b.h, "y")
    close(h_last, last, b.h, "h_last")
    if not backward:
        return
    dy = layout(kind, T, E, H, dtype, normal(T, E, H))[0]
    dl = normal(E, H) if dh_last else None
    df, dx, dh0, dbias = hip.glr_backward(a["f"], a["x"], dy, saved, resets=a["resets"], bias=a["bias"], dh_last=dl)
    wf, wx, w0, wb = ref.backward(a["f"], a["x"], a["h0"], a["resets"], a["bias"], dy, dl)
    tg, tx, tf = b.grads(ref.largest_g(a["f"], a["bias"], a["resets"], dy, dl))
    close(df, wf, tf, "df")
    close(dx, wx, tx, "dx")
    close(dh0, w0, tg, "dh0")
    if a["bias"] is None:
        assert dbias is None
    else:
        # every term's own error, and float32 sums of at most 64 terms in a row (64 U of the terms' sizes) before they widen
        close(dbias, wb, T * tf.sum(0) + 64 * ref.U * wf.abs().sum((0, 1)) + ref.U * wb.abs(), "dbias")


SIZES = [(1, 1, 1), (1, 37, 333), (2, 3, 5), (15, 2, 64), (16, 1, 128), (17, 4, 65), (31, 1, 200), (33, 5, 7), (64, 1, 1), (100, 3, 130),
         (255, 2, 96), (256, 1, 64), (257, 2, 64), (513, 2, 70), (1001, 7, 33), (2049, 1, 258), (5000, 1, 64), (3, 300, 256), (128, 64, 256),
         (40, 1, 2048), (777, 1, 1000), (9001, 1, 70), (12293, 2, 33), (4096, 1, 64), (4097, 3, 50), (300, 200, 256)]


@pytest.mark.parametrize("T,E,H", SIZES)
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_sizes(hip, T, E, H, dtype):
    k = T + E + H
    a, normal = make(T, E, H, dtype, resets=k % 2 == 0, bias=k % 3 != 0, h0=k % 5 != 0, seed=k)
    check(hip, a, normal, dtype)


@pytest.mark.parametrize("kind", ["joint", "batch first", "odd"])
@pytest.mark.parametrize("T,E,H", [(70, 3, 64), (300, 2, 129), (19, 33, 256), (1, 5, 130)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_layouts(hip, kind, T, E, H, dtype):
    a, normal = make(T, E, H, dtype, kind=kind, resets=True, bias=True, seed=T)
    if kind == "batch first":
        a["resets"] = a["resets"].t().contiguous().t()
    check(hip, a, normal, dtype, kind)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,E,H", [(300, 2, 129), (20, 3, 64)])
def test_outputs_into_views_leave_the_rest_alone(hip, dtype, T, E, H):
    a, normal = make(T, E, H, dtype, resets=True, bias=True)
    y, ybuf = layout("odd", T, E, H, dtype, None)
    ybuf.fill_(7.0)
    keep = torch.ones_like(ybuf, dtype=torch.bool)
    keep[3:].as_strided(y.shape, y.stride(), 3).fill_(False)
    hbuf = torch.full((E + 2, H), 7.0, device="cuda")
    want, last, saved = hip.glr_forward(a["f"], a["x"], a["h0"], resets=a["resets"], bias=a["bias"], want_saved=True)
    got = hip.glr_forward(a["f"], a["x"], a["h0"], resets=a["resets"], bias=a["bias"], y=y, h_last=hbuf[1:E + 1])
    assert got[0] is y and got[2] is None
    assert torch.equal(y, want) and torch.equal(hbuf[1:E + 1], last)
    assert bool((ybuf[keep] == 7.0).all()) and bool((hbuf[0] == 7).all()) and bool((hbuf[E + 1] == 7).all())
    dy = normal(T, E, H).to(dtype)
    wf, wx, w0, wb = hip.glr_backward(a["f"], a["x"], dy, saved, resets=a["resets"], bias=a["bias"])
    joint = torch.full((T + 1, E, 2 * H), 7.0, dtype=dtype, device="cuda")
    df, dx, d0, db = hip.glr_backward(a["f"], a["x"], dy, saved, resets=a["resets"], bias=a["bias"], df=joint[:T, :, :H], dx=joint[:T, :, H:])
    assert torch.equal(joint[:T, :, :H], wf) and torch.equal(joint[:T, :, H:], wx) and bool((joint[T] == 7).all())
    assert torch.equal(d0, w0) and torch.equal(db, wb)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_broadcast_inputs(hip, dtype):
    T, E, H = 50, 6, 96
    a, normal = make(T, E, H, dtype, bias=True)
    a["f"] = a["f"][:, :1].expand(T, E, H)          # one gate for all envs
    a["x"] = a["x"][:1].expand(T, E, H)             # one input for all steps
    a["resets"] = (torch.rand(T, 1, device="cuda") < 0.1).expand(T, E)
    check(hip, a, normal, dtype)


@pytest.mark.parametrize("T", [1, 40, 700])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_masks_that_leave_nothing(hip, T, dtype):
    a, normal = make(T, 3, 70, dtype, bias=True)
    a["resets"] = torch.zeros(T, 3, dtype=torch.bool, device="cuda")
    a["resets"][:, 0] = True                        # a state that never survives
    a["resets"][0, 1] = True
    check(hip, a, normal, dtype)


@pytest.mark.parametrize("T", [5, 40, 700, 9000])
def test_what_a_reset_hides_has_no_influence(hip, T):
    """A first state and inputs that are not numbers, in front of a reset: nothing of them behind it, in either direction."""
    E, H, r = 2, 70, T // 2
    a, normal = make(T, E, H, F32, bias=True)
    a["resets"] = torch.zeros(T, E, dtype=torch.uint8, device="cuda")
    a["resets"][r] = 3                              # any value but zero is a flag
    dy = normal(T, E, H)
    clean = hip.glr_forward(a["f"], a["x"], a["h0"], resets=a["resets"], bias=a["bias"], want_saved=True)
    gclean = hip.glr_backward(a["f"], a["x"], dy, clean[2], resets=a["resets"], bias=a["bias"])
    for bad in (float("nan"), float("inf"), -float("inf")):
        h0, x = a["h0"].clone(), a["x"].clone()
        h0[0, 3] = bad
        x[r - 1, 1, 5] = bad
        y, last, saved = hip.glr_forward(a["f"], x, h0, resets=a["resets"], bias=a["bias"], want_saved=True)
        assert torch.equal(y[r:], clean[0][r:]) and torch.equal(last, clean[1])
        assert not bool(torch.isfinite(y[:r, 0, 3]).any()) and not bool(torch.isfinite(y[r - 1, 1, 5]))
        rest = torch.ones_like(y, dtype=torch.bool)
        rest[:r, 0, 3] = False
        rest[:r, 1, 5] = False
        assert torch.equal(y[rest], clean[0][rest])
        dyb = dy.clone()
        dyb[r, 1, 9] = bad                          # and a gradient behind the reset does not reach in front of it
        df, dx, dh0, _ = hip.glr_backward(a["f"], x, dyb, saved, resets=a["resets"], bias=a["bias"])
        assert torch.equal(dx[:r], gclean[1][:r]) and torch.equal(dh0, gclean[2])
        assert torch.equal(df[r + 1:], gclean[0][r + 1:])
    # a reset at the first step hides h0 as a whole
    a["resets"][0] = 1
    y0, _, s0 = hip.glr_forward(a["f"], a["x"], torch.full_like(a["h0"], float("nan")), resets=a["resets"], bias=a["bias"], want_saved=True)
    assert bool(torch.isfinite(y0).all())
    df, dx, dh0, db = hip.glr_backward(a["f"], a["x"], dy, s0, resets=a["resets"], bias=a["bias"])
    assert bool((dh0 == 0).all()) and bool(torch.isfinite(df).all()) and bool(torch.isfinite(db).all())


@pytest.mark.parametrize("T", [3, 50, 600])
def test_gates_at_their_ends(hip, T):
    """Gates that are fully open or shut, by infinities, by the type's ends and by sizes where exp leaves float32."""
    ends = [float("inf"), -float("inf"), 3.4028234e38, -3.4028234e38, 200.0, -200.0, 90.0, -90.0, 30.0, -30.0, 17.0, -17.0, 0.0]
    f = torch.tensor(ends, device="cuda").expand(T, 2, len(ends)).contiguous()
    g = torch.Generator(device="cuda").manual_seed(1)
    x, dy = (torch.randn(f.shape, generator=g, device="cuda") for _ in range(2))
    h0 = torch.randn(2, len(ends), generator=g, device="cuda")
    y, last, saved = hip.glr_forward(f, x, h0, want_saved=True)
    want = ref.forward(f, x, h0)[0]
    # worst case of the size of glr_reference.Bounds with K = T and gates 8 U off; f itself is exact here
    tol = ref.U * 4.0 * (16 + 6 * T)
    close(y, want, torch.full_like(want, tol), "y")
    assert torch.equal(y[:, :, 0], h0[:, 0].expand(T, 2)) and torch.equal(y[:, :, 1], x[:, :, 1])
    df, dx, dh0, _ = hip.glr_backward(f, x, dy, saved)
    wf, wx, w0, _ = ref.backward(f, x, h0, None, None, dy)
    top = ref.largest_g(f, None, None, dy, None)
    tol = ref.U * top * (64 + 6 * T)
    close(dx, wx, tol, "dx")
    close(df, wf, 4 * tol, "df")
    close(dh0, w0, tol, "dh0")


@pytest.mark.parametrize("T", [4, 40, 600, 9000])
def test_infinities_and_nans_follow_the_formula(hip, T):
    f = torch.zeros(T, 1, 8, device="cuda")
    x = torch.ones(T, 1, 8, device="cuda")
    x[1, 0, 0], x[1, 0, 1], x[1, 0, 2] = float("inf"), -float("inf"), float("nan")
    x[1, 0, 3], x[2, 0, 3] = float("inf"), -float("inf")
    f[2, 0, 4] = float("nan")
    x[1, 0, 5], x[2, 0, 5] = 3e38, -3e38            # a distance beyond float32
    f[:, 0, 6] = 4.0
    x[1, 0, 6] = float("inf")                       # kept by a gate next to one
    f[:, 0, 7] = -4.0
    x[1, 0, 7] = float("inf")
    y, last, _ = hip.glr_forward(f, x)
    want = ref.forward(f, x)[0].float()
    assert torch.equal(torch.isnan(y), torch.isnan(want)) and torch.equal(torch.isinf(y), torch.isinf(want))
    fin = torch.isfinite(want)
    assert torch.equal(torch.sign(y[~fin & ~torch.isnan(want)]), torch.sign(want[~fin & ~torch.isnan(want)]))
    assert bool(((y[fin] - want[fin]).abs() <= 1e-5 * want[fin].abs() + 1e-5).all())        # K = 2: 28 U of the largest input of the column


def test_long_memory(hip):
    """Gates of 1 - 3e-6 over 20000 steps: a gate rounded to float32 would be off by 1 % of its distance to one.  The bound
    counts one rounding of the state per span of 16 steps at random signs, not one per step: a straight sum of the worst case
    says 20000 U = 1e-3, which the rounded gate would pass as well."""
    T, H = 20000, 64
    g = torch.Generator(device="cuda").manual_seed(2)
    f = torch.full((T, 1, H), 12.7, device="cuda")
    x = 1 + 0.1 * torch.randn(T, 1, H, generator=g, device="cuda")
    y, last, saved = hip.glr_forward(f, x, want_saved=True)
    want = ref.forward(f, x)[0]
    rel = ((y.double() - want).abs().amax((1, 2)) / want.abs().amax((1, 2)))[100:]
    # 20000 roundings of at most U each, all the same way, against a state that grows to 6 %: 20000 U * (sum of the states so far
    # over steps and the last state) <= 20000 U / 2 = 6e-4; at random signs sqrt(20000) U = 8.4e-6, six times that for the worst of 64 columns
    assert float(rel.max()) < 5.1e-5, float(rel.max())
    dy = torch.randn(T, 1, H, generator=g, device="cuda")
    df, dx, dh0, _ = hip.glr_backward(f, x, dy, saved)
    wf, wx, w0, _ = ref.backward(f, x, None, None, None, dy)
    for got, w in ((df, wf), (dx, wx), (dh0, w0)):
        assert float((got.double() - w).norm() / w.norm()) < 5.1e-5


def test_nothing_to_do(hip):
    z = lambda *s: torch.zeros(s, device="cuda")        # noqa: E731
    h0 = torch.randn(3, 5, device="cuda")
    y, last, saved = hip.glr_forward(z(0, 3, 5), z(0, 3, 5), h0, bias=z(5), want_saved=True)
    assert y.shape == (0, 3, 5) and torch.equal(last, h0)
    dl = torch.randn(3, 5, device="cuda")
    df, dx, dh0, db = hip.glr_backward(z(0, 3, 5), z(0, 3, 5), z(0, 3, 5), saved, bias=z(5), dh_last=dl)
    assert torch.equal(dh0, dl) and bool((db == 0).all()) and df.shape == (0, 3, 5)
    assert bool((hip.glr_forward(z(0, 3, 5), z(0, 3, 5))[1] == 0).all())
    for shape in ((4, 0, 5), (4, 3, 0)):
        y, last, saved = hip.glr_forward(z(*shape), z(*shape), bias=z(shape[2]), want_saved=True)
        assert y.shape == shape and last.shape == shape[1:]
        df, dx, dh0, db = hip.glr_backward(z(*shape), z(*shape), z(*shape), saved, bias=z(shape[2]))
        assert db.shape == (shape[2],) and bool((db == 0).all())
    assert hip.glr_step(z(0, 5), z(0, 5), z(0, 5)).shape == (0, 5)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_steps_follow_the_sequence(hip, dtype):
    T, E, H = 40, 37, 129
    a, _ = make(T, E, H, dtype, kind="joint", resets=True, bias=True)
    want, last, _ = ref.forward(a["f"], a["x"], a["h0"], a["resets"], a["bias"])
    tol = ref.Bounds(a["f"], a["x"], a["h0"], a["resets"], a["bias"]).h
    state = a["h0"].clone()
    out = torch.empty(E, H, dtype=dtype, device="cuda")
    for t in range(T):
        y = hip.glr_step(a["f"][t], a["x"][t], state, resets=a["resets"][t], bias=a["bias"], y=out if t % 2 else None)
        assert (y is out) == bool(t % 2)
        close(y, want[t], tol, "y[%d]" % t)
    close(state, last, tol, "state")


def test_state_may_be_none_of_the_outputs(hip):
    s = torch.zeros(3, 8, device="cuda")
    with pytest.raises(ValueError, match="overlaps"):
        hip.glr_step(torch.zeros(3, 8, device="cuda"), torch.zeros(3, 8, device="cuda"), s, y=s)
    with pytest.raises(ValueError, match="overlaps"):
        hip.glr_forward(torch.zeros(2, 3, 8, device="cuda"), torch.zeros(2, 3, 8, device="cuda"), h0=s, h_last=s)
    with pytest.raises(TypeError, match="all tensors"):
        hip.glr_forward(torch.zeros(2, 3, 8), torch.zeros(2, 3, 8, device="cuda"))


@pytest.mark.parametrize("T,E,H", [(600, 2, 130), (20000, 1, 64), (20, 300, 64), (40, 200, 256)])
def test_same_bits_every_time(hip, T, E, H):
    a, normal = make(T, E, H, BF16, resets=True, bias=True)
    dy = normal(T, E, H).to(BF16)
    first = None
    for _ in range(3):
        y, last, saved = hip.glr_forward(a["f"], a["x"], a["h0"], resets=a["resets"], bias=a["bias"], want_saved=True)
        out = (y, last) + hip.glr_backward(a["f"], a["x"], dy, saved, resets=a["resets"], bias=a["bias"])
        first = first or out
        assert all(torch.equal(p, q) for p, q in zip(first, out))


def test_gradients_against_differences(hip):
    """Directional differences of the GPU's own forward pass, summed in 64 bits: step 2^-7 leaves 6e-5 times third derivatives of
    order one of a loss of 2000 terms at random signs, and float32 values of 2^-24 * 40 per term over the step."""
    T, E, H = 50, 2, 20
    a, normal = make(T, E, H, F32, bias=True, reach=2.0)
    w, wl = normal(T, E, H), normal(E, H)

    def loss(f, x, h0, b):
        y, last, _ = hip.glr_forward(f, x, h0, bias=b)
        return float((y.double() * w).sum() + (last.double() * wl).sum())

    _, _, saved = hip.glr_forward(a["f"], a["x"], a["h0"], bias=a["bias"], want_saved=True)
    df, dx, dh0, db = hip.glr_backward(a["f"], a["x"], w, saved, bias=a["bias"], dh_last=wl)
    at = [a["f"], a["x"], a["h0"], a["bias"]]
    for k, grad in enumerate((df, dx, dh0, db)):
        v = torch.randn_like(at[k])
        v /= v.norm()
        up, down = ([q + s * v if i == k else q for i, q in enumerate(at)] for s in (2.0 ** -7, -2.0 ** -7))
        diff = (loss(*up) - loss(*down)) * 2.0 ** 6
        want = float((grad.double() * v).sum())
        assert abs(diff - want) < 2e-2 * (1 + abs(want)), (k, diff, want)


@pytest.mark.parametrize("T,E,H", [(6000, 3, 200), (30, 200, 256)])
def test_another_stream(hip, T, E, H):
    a, normal = make(T, E, H, BF16, resets=True, bias=True)
    dy = normal(T, E, H).to(BF16)
    want = hip.glr_forward(a["f"], a["x"], a["h0"], resets=a["resets"], bias=a["bias"], want_saved=True)
    gwant = hip.glr_backward(a["f"], a["x"], dy, want[2], resets=a["resets"], bias=a["bias"])
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = []
    for s in (s1, s2, s1, s2):                     # calls that overlap in time share nothing
        with torch.cuda.stream(s):
            y, last, saved = hip.glr_forward(a["f"], a["x"], a["h0"], resets=a["resets"], bias=a["bias"], want_saved=True)
            outs.append((y, last) + hip.glr_backward(a["f"], a["x"], dy, saved, resets=a["resets"], bias=a["bias"]))
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(p, q) for p, q in zip(o, want[:2] + gwant))


@pytest.mark.parametrize("T,E,H", [(9000, 1, 128), (40, 4, 64), (30, 200, 256)])
def test_captured_and_replayed(hip, T, E, H):
    """Two graphs with their own workspaces, replayed in turn with eager work between, against eager results on new inputs."""
    a, normal = make(T, E, H, F32, resets=True, bias=True)
    dy = normal(T, E, H)
    one = lambda: hip.glr_forward(a["f"], a["x"], a["h0"], resets=a["resets"], bias=a["bias"], want_saved=True)       # noqa: E731

    def both():
        y, last, saved = one()
        return (y, last) + hip.glr_backward(a["f"], a["x"], dy, saved, resets=a["resets"], bias=a["bias"])
    both()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = both()
        graphs.append((g, outs))
    for k in range(4):
        for t in (a["f"], a["x"], a["h0"], dy):
            t.copy_(torch.randn_like(t))
        a["resets"].copy_(torch.rand(T, E, device="cuda") < 0.1)
        want = both()
        for g, outs in graphs:
            for o in outs:
                o.fill_(3.0)
            g.replay()
        graphs[k % 2][0].replay()
        torch.cuda.synchronize()
        for g, outs in graphs:
            assert all(torch.equal(p, q) for p, q in zip(outs, want)), k


def test_envs_far_apart(hip):
    """Envs 2^28 elements apart: a tile's lanes no longer reach them with 32-bit offsets."""
    T, E, H = 300, 3, 34
    se = 1 << 28
    buf = torch.empty((E - 1) * se + T * H * 2 + 8, dtype=BF16, device="cuda")
    views = [buf.as_strided((T, E, H), (2 * H, se, 1), k * H) for k in range(2)]
    a, normal = make(T, E, H, BF16, resets=True, bias=True)
    for v, t in zip(views, (a["f"], a["x"])):
        v.copy_(t)
    a["f"], a["x"] = views
    check(hip, a, normal, BF16)
    t, _ = make(20, E, H, BF16)
    for v, w in zip(views, (t["f"], t["x"])):
        v[:20].copy_(w)
    a["f"], a["x"], a["resets"] = views[0][:20], views[1][:20], None
    check(hip, a, normal, BF16)


def test_offsets_beyond_32_bits(hip):
    """Steps 2^31 + 40 elements apart (a bfloat16 buffer of 12.9 GB of which three rows are used)."""
    T, E, H = 3, 2, 70
    st = (1 << 31) + 40
    buf = torch.empty((T - 1) * st + 400, dtype=BF16, device="cuda")
    views = [buf.as_strided((T, E, H), (st, H, 1), k * 140) for k in range(2)]
    a, normal = make(T, E, H, BF16, bias=True)
    for v, t in zip(views, (a["f"], a["x"])):
        v.copy_(t)
    a["f"], a["x"] = views
    check(hip, a, normal, BF16)


_GAVE_UP_SCRIPT = """
import sys
sys.path.insert(0, sys.argv[1])
import torch
from baselines_amd import _lib, hip
T, E, H = 700, 2, 70
f, x, dy = (torch.randn(T, E, H, device="cuda") for _ in range(3))
seen = []
def look(what):
    torch.cuda.synchronize()
    try:
        hip.take_faults()
    except _lib.Ppo2HipError as e:
        seen.append(what + ": " + str(e))
y, _, saved = hip.glr_forward(f, x, want_saved=True)
look("forward")
hip.glr_backward(f, x, dy, saved)
look("backward")
hip.glr_forward(f[:256], x[:256])
look("held")
print("SEEN", len(seen), seen)
"""


@pytest.mark.parametrize("forced", [False, True])
def test_a_chain_that_gave_up_is_reported(tmp_path, forced):
    """PPO2HIP_GRID_SYNC_SPINS=-1 makes every wait of the chain count as given up: both long passes raise the library's fault word
    and end as usual, and a sequence that one workgroup holds, which waits for nobody, raises nothing."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    script = tmp_path / "gave_up.py"
    script.write_text(_GAVE_UP_SCRIPT)
    env = dict(os.environ)
    if forced:
        env["PPO2HIP_GRID_SYNC_SPINS"] = "-1"
    res = subprocess.run([sys.executable, str(script), root], env=env, capture_output=True, text=True, timeout=100)
    assert res.returncode == 0, res.stderr[-2000:]
    line = [l for l in res.stdout.splitlines() if l.startswith("SEEN")][0]
    assert line.startswith("SEEN 2" if forced else "SEEN 0"), line
    assert not forced or ("forward" in line and "backward" in line and "gave up" in line)


@pytest.mark.parametrize("T,E,H", [(1, 4100, 33), (2, 2049, 1), (300, 70, 65)])
def test_bias_gradient_over_many_rows(hip, T, E, H):
    """More rows of partial sums than one workgroup adds up, and columns that end inside a workgroup's 32."""
    a, normal = make(T, E, H, F32, bias=True, seed=E)
    check(hip, a, normal, F32)


def test_several_calls_at_once(hip):
    """Chains of workgroups on four streams at a time: each hands on its own states and none waits for another."""
    sizes = [(9000, 2, 130), (4000, 3, 257), (20000, 1, 96), (2100, 8, 200)]
    calls = []
    for i, (T, E, H) in enumerate(sizes):
        a, normal = make(T, E, H, (F32, BF16)[i % 2], resets=True, bias=True, seed=i)
        calls.append((a, normal(T, E, H).to(a["x"].dtype), torch.cuda.Stream()))

    def both(a, dy):
        y, last, saved = hip.glr_forward(a["f"], a["x"], a["h0"], resets=a["resets"], bias=a["bias"], want_saved=True)
        return (y, last) + hip.glr_backward(a["f"], a["x"], dy, saved, resets=a["resets"], bias=a["bias"])
    want = [both(a, dy) for a, dy, _ in calls]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for a, dy, s in calls:
            with torch.cuda.stream(s):
                got.append(both(a, dy))
    torch.cuda.synchronize()
    hip.take_faults()
    for k, outs in enumerate(got):
        assert all(torch.equal(p, q) for p, q in zip(outs, want[k % len(calls)])), k


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_long_16_bit_sequences(hip, dtype):
    """Over several blocks of batches, 128 * 64 steps each, with a reset now and then in one env only."""
    T, E, H = 17000, 2, 66
    a, normal = make(T, E, H, dtype, bias=True, seed=5)
    a["resets"] = torch.zeros(T, E, dtype=torch.bool, device="cuda")
    a["resets"][[0, 8191, 8192, 16390], 1] = True
    check(hip, a, normal, dtype)


def _relative(share, each, back=False):
    """Relative error of a scan whose terms are all positive, step by step: what came over by its share of the step's value, and
    `each` for the step itself."""
    r, out = torch.zeros_like(share[0]), torch.empty_like(share)
    for t in range(share.shape[0] - 1, -1, -1) if back else range(share.shape[0]):
        r = share[t] * r + each
        out[t] = r
    return out


@pytest.mark.parametrize("T", [1, 5, 40, 300, 9000])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_gates_almost_shut_keep_their_share(hip, T, dtype):
    """States of 1e4 behind gates of 1e-8 beside inputs of 1e-3, and gradients likewise.  Every term is positive, so errors stay
    relative: a gate's (8 + 2 Z) U, two products, the sum, and three roundings where runs are joined, twice that for good measure."""
    E, H, z = 2, 70, 18.375
    g = torch.Generator(device="cuda").manual_seed(T)
    kind = torch.rand((T, E, H), generator=g, device="cuda")
    f = torch.where(kind < 0.6, -z, torch.where(kind < 0.8, 0.0, 3.0)).to(dtype)
    x = (torch.where((kind >= 0.6) & (kind < 0.8), 1e4, 1e-3) * (0.5 + torch.rand((T, E, H), generator=g, device="cuda"))).to(dtype)
    h0 = 1e4 * (0.5 + torch.rand((E, H), generator=g, device="cuda"))
    y, last, saved = hip.glr_forward(f, x, h0, want_saved=True)
    want, wlast, ps = ref.forward(f, x, h0)
    each = (20 + 2 * z) * ref.U
    a = torch.sigmoid(f.double())
    rel = _relative(a * ps / want, each)
    close(y, want, rel * want, "y")
    close(last, wlast, rel[-1] * wlast, "h_last")
    kind = torch.rand((T, E, H), generator=g, device="cuda")
    dy = (torch.where(kind < 0.3, 1e4, 1e-3) * (0.5 + torch.rand((T, E, H), generator=g, device="cuda"))).to(dtype)
    dl = 1e4 * (0.5 + torch.rand((E, H), generator=g, device="cuda"))
    _, dx, dh0, _ = hip.glr_backward(f, x, dy, saved, dh_last=dl)
    _, wx, w0, _ = ref.backward(f, x, h0, None, None, dy, dl)
    om = torch.sigmoid(-f.double())
    rel = _relative(1 - dy.double() * om / wx, each, back=True)
    close(dx, wx, (rel + each) * wx, "dx")
    close(dh0, w0, (rel[0] + each) * w0, "dh0")



_FAR = [-17.0, -30.0, -60.0, -88.0, -100.0, -110.0, -300.0, -700.0, 17.0, 60.0, 86.0, 0.5, 88.0, 110.0, 300.0, 700.0]


@pytest.mark.parametrize("T", [1, 5, 40, 600, 9000])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_infinite_states_pass_every_gate(hip, T, dtype):
    """sigmoid of a finite number is not zero: an infinite state, input or gradient stays one however far the gate, in the span that
    it enters and in all that follow.  The definition makes it no number at a gate of minus infinity, and 1 - a of a gate beyond 87 is
    zero in the hardware's exponent: what is left there is not finite either way."""
    H = len(_FAR)
    f = torch.tensor(_FAR, device="cuda").to(dtype).expand(T, 4, H).contiguous()
    g = torch.Generator(device="cuda").manual_seed(T)
    x, dy = ((0.5 + torch.rand((T, 4, H), generator=g, device="cuda")).to(dtype) for _ in range(2))
    h0 = 0.5 + torch.rand(4, H, generator=g, device="cuda")
    h0[0] = float("inf")                            # env 0 begins so, env 1 meets an infinity on the way, env 2 a shut gate behind one
    x[T // 3, 1, :12] = -float("inf")
    h0[2] = -float("inf")
    f[T // 2, 2] = -float("inf")
    dl = torch.ones(4, H, device="cuda")
    dl[0] = float("inf")
    dy[(2 * T) // 3, 1] = float("inf")
    y, last, saved = hip.glr_forward(f, x, h0, want_saved=True)
    want, wlast, _ = ref.forward(f, x, h0)
    df, dx, dh0, _ = hip.glr_backward(f, x, dy, saved, dh_last=dl)
    _, wx, w0, _ = ref.backward(f, x, h0, None, None, dy, dl)
    for name, got, w in (("y", y, want), ("h_last", last, wlast), ("dx", dx, wx), ("dh0", dh0, w0)):
        assert torch.equal(torch.isfinite(got), torch.isfinite(w)), name
        sure = torch.isinf(w)                       # infinite by the definition
        if name == "dx":
            sure[:, :, 12:] = False
        assert torch.equal(got[sure].double(), w[sure]), name
        fin = torch.isfinite(w)
        # at most T steps of (20 + 2 Z) U of values of at most 3/2 (g: at most T of them and the last), and half a step of the type
        top = 1.5 if name in ("y", "h_last") else 1.5 * T + 1
        tol = (20 + 2 * 700) * T * ref.U * top + half_step(got.dtype) * w[fin].abs()
        assert bool(((got[fin].double() - w[fin]).abs() <= tol).all()), name


@pytest.mark.parametrize("T", [5, 40, 700, 9000])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("E,H", [(2, 70), (3, 33)])
def test_what_a_reset_hides_in_16_bits(hip, T, dtype, E, H):
    """What is not finite stays in its own column, and in front of the reset, bit for bit, in both directions."""
    r = T // 2
    a, normal = make(T, E, H, dtype, bias=True)
    a["resets"] = torch.zeros(T, E, dtype=torch.uint8, device="cuda")
    a["resets"][r] = 1
    dy = normal(T, E, H).to(dtype)
    clean = hip.glr_forward(a["f"], a["x"], a["h0"], resets=a["resets"], bias=a["bias"], want_saved=True)
    gclean = hip.glr_backward(a["f"], a["x"], dy, clean[2], resets=a["resets"], bias=a["bias"])
    for bad in (float("nan"), float("inf"), -float("inf")):
        h0, x = a["h0"].clone(), a["x"].clone()
        h0[0, 3] = bad
        x[r - 1, 1, 5] = bad
        y, last, saved = hip.glr_forward(a["f"], x, h0, resets=a["resets"], bias=a["bias"], want_saved=True)
        assert torch.equal(y[r:], clean[0][r:]) and torch.equal(last, clean[1])
        assert not bool(torch.isfinite(y[:r, 0, 3]).any()) and not bool(torch.isfinite(y[r - 1, 1, 5]))
        rest = torch.ones_like(y, dtype=torch.bool)
        rest[:r, 0, 3] = False
        rest[r - 1, 1, 5] = False
        assert torch.equal(y[rest], clean[0][rest])
        dyb = dy.clone()
        dyb[r, 1, 9] = bad
        df, dx, dh0, _ = hip.glr_backward(a["f"], x, dyb, saved, resets=a["resets"], bias=a["bias"])
        assert torch.equal(dx[:r], gclean[1][:r]) and torch.equal(dh0, gclean[2])
        assert torch.equal(df[r + 1:], gclean[0][r + 1:])


_GAVE_UP_VALUES_SCRIPT = """
import sys
sys.path.insert(0, sys.argv[1])
import torch
from baselines_amd import hip
for dt in (torch.float32, torch.bfloat16):
    T, E, H = 700, 2, 70
    f, x, dy = (torch.randn(T, E, H, device="cuda").to(dt) for _ in range(3))
    y, last, saved = hip.glr_forward(f, x, want_saved=True)
    df, dx, dh0, _ = hip.glr_backward(f, x, dy, saved)
    hip.take_faults(raise_on_fault=False)
    ok = bool(torch.isfinite(y[:128]).all()) and bool(torch.isnan(y[128:]).all()) and bool(torch.isnan(last).all())
    ok = ok and bool(torch.isfinite(dx[640:]).all()) and bool(torch.isnan(dx[:640]).all()) and bool(torch.isnan(dh0).all())
    print("VALUES", ok)
"""


def test_a_chain_that_gave_up_leaves_nan(tmp_path):
    """Behind the batch of 128 steps that waits for nobody nothing looks like a result, whatever had been published by then."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    script = tmp_path / "gave_up.py"
    script.write_text(_GAVE_UP_VALUES_SCRIPT)
    env = dict(os.environ, PPO2HIP_GRID_SYNC_SPINS="-1")
    res = subprocess.run([sys.executable, str(script), root], env=env, capture_output=True, text=True, timeout=100)
    assert res.returncode == 0, res.stderr[-2000:]
    assert [l for l in res.stdout.splitlines() if l.startswith("VALUES")] == ["VALUES True"] * 2, res.stdout


@pytest.mark.parametrize("dtype", [F32, F16])
def test_steps_over_windows(hip, dtype):
    """Inputs whose rows overlap: every env a window of one row, a step along; outputs have rows of their own."""
    E, H = 5, 70
    row = torch.randn(2, E + H, device="cuda").to(dtype)
    f, x = (row[k].as_strided((E, H), (1, 1)) for k in range(2))
    state = torch.randn(E, H, device="cuda")
    want = ref.forward(f.unsqueeze(0), x.unsqueeze(0), state)[0][0]
    tol = ref.Bounds(f.unsqueeze(0), x.unsqueeze(0), state, None, None).h
    y = hip.glr_step(f, x, state)
    assert y.is_contiguous()
    close(y, want, tol, "y")
    close(state, want, tol, "state")
    y, last, _ = hip.glr_forward(f.expand(3, E, H), x.expand(3, E, H))
    want = ref.forward(f.expand(3, E, H), x.expand(3, E, H))[0]
    close(y, want, 3 * tol, "sequence")


def walks_back(hip, dtype, E, H):
    """Whether the gradients of so many columns go back with one wave per tile: a long sequence then needs no workspace."""
    from baselines_amd import _lib
    return _lib.lib.ppo2hip_glr_backward_workspace_bytes(hip._GLR_TYPES[dtype], 300, E, H, 0) == 0


@pytest.mark.parametrize("T,E,H,kind", [(1, 2500, 33, "apart"), (16, 1300, 64, "apart"), (17, 640, 129, "joint"), (40, 330, 256, "batch first"), (300, 330, 250, "apart"),
                                        (270, 2, 41000, "odd"), (33, 81920, 1, "apart")])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_many_columns_in_16_bits(hip, T, E, H, kind, dtype):
    """Gradients that a wave walks back by itself over all steps of its columns, from one span to many, the last one cut short."""
    assert walks_back(hip, dtype, E, H)
    k = T + E + H
    a, normal = make(T, E, H, dtype, kind=kind, resets=k % 2 == 0, bias=k % 3 != 0, h0=k % 5 != 0, seed=k)
    check(hip, a, normal, dtype, kind, dh_last=k % 7 != 0)
    if a["bias"] is None or a["resets"] is None:
        a, normal = make(T, E, H, dtype, kind=kind, resets=True, bias=True, seed=k)
        check(hip, a, normal, dtype, kind)


@pytest.mark.parametrize("T", [5, 40, 300])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_what_a_reset_hides_from_many_columns(hip, T, dtype):
    E, H, r = 3, 27500, T // 2
    assert walks_back(hip, dtype, E, H)
    a, normal = make(T, E, H, dtype, bias=True)
    a["resets"] = torch.zeros(T, E, dtype=torch.uint8, device="cuda")
    a["resets"][r] = 1
    dy = normal(T, E, H).to(dtype)
    clean = hip.glr_forward(a["f"], a["x"], a["h0"], resets=a["resets"], bias=a["bias"], want_saved=True)
    gclean = hip.glr_backward(a["f"], a["x"], dy, clean[2], resets=a["resets"], bias=a["bias"])
    for bad in (float("nan"), float("inf"), -float("inf")):
        h0, x, dyb = a["h0"].clone(), a["x"].clone(), dy.clone()
        h0[0, 3] = bad
        x[r - 1, 1, 5] = bad
        dyb[r, 2, H - 1] = bad
        y, last, saved = hip.glr_forward(a["f"], x, h0, resets=a["resets"], bias=a["bias"], want_saved=True)
        assert torch.equal(y[r:], clean[0][r:]) and torch.equal(last, clean[1])
        df, dx, dh0, _ = hip.glr_backward(a["f"], x, dyb, saved, resets=a["resets"], bias=a["bias"])
        assert torch.equal(dx[:r], gclean[1][:r]) and torch.equal(dh0, gclean[2])
        assert torch.equal(df[r + 1:], gclean[0][r + 1:])
        rest = torch.ones_like(df, dtype=torch.bool)
        rest[:r, 0, 3] = False
        rest[:r, 1, 5] = False
        rest[r, 2, H - 1] = False
        assert torch.equal(df[rest], gclean[0][rest])


def test_many_columns_of_envs_far_apart(hip):
    """Envs 2^29 elements apart: each has tiles of its own, the last one of 40 columns."""
    T, E, H = 20, 2, 41000
    se = 1 << 29
    assert walks_back(hip, BF16, E, H)
    buf = torch.empty((E - 1) * se + T * H * 2 + 8, dtype=BF16, device="cuda")
    views = [buf.as_strided((T, E, H), (2 * H, se, 1), k * H) for k in range(2)]
    a, normal = make(T, E, H, BF16, resets=True, bias=True)
    for v, t in zip(views, (a["f"], a["x"])):
        v.copy_(t)
    a["f"], a["x"] = views
    check(hip, a, normal, BF16)


@pytest.mark.parametrize("T", [20, 300])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_gates_around_one_half(hip, T, dtype):
    """f + bias at and next to zero, from either side, where a gate is held by its other side: a run of such gates between two that
    keep everything, and runs with only one of them."""
    near = [0.0, -0.0, 2.0 ** -24, -2.0 ** -24, 3e-7, -3e-7, 1e-5, -1e-5, 2.0 ** -120, -2.0 ** -120, 0.7, -0.7, 1.1, 1.09]
    bias = torch.tensor(near, device="cuda")
    f = torch.full((T, 3, len(near)), 40.0, device="cuda").to(dtype)
    f[5, 0] = 0.0                                   # one gate of the span
    f[3:17, 1] = 0.0
    f[:, 2] = 0.0
    g = torch.Generator(device="cuda").manual_seed(T)
    x, dy = (torch.randn(f.shape, generator=g, device="cuda").to(dtype) for _ in range(2))
    h0 = torch.randn(3, len(near), generator=g, device="cuda")
    check(hip, dict(f=f, x=x, h0=h0, resets=None, bias=bias), lambda *s: torch.randn(s, generator=g, device="cuda"), dtype)


@pytest.mark.parametrize("T,E,H", [(9000, 2, 70), (100, 30, 70)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_a_column_that_is_no_number_changes_no_other(hip, T, E, H, dtype):
    """A wave that walks a span the slow way for one of its columns rounds the others' outputs as the quick way does."""
    a, normal = make(T, E, H, dtype, bias=True)
    dy = normal(T, E, H).to(dtype)

    def both(x, dy):
        y, last, saved = hip.glr_forward(a["f"], x, a["h0"], bias=a["bias"], want_saved=True)
        return (y, last) + hip.glr_backward(a["f"], x, dy, saved, bias=a["bias"])
    clean = both(a["x"], dy)
    x, dyb = a["x"].clone(), dy.clone()
    x[1, 1, 5], dyb[T - 2, 0, 9] = float("nan"), float("inf")
    got = both(x, dyb)
    ok = torch.ones(E, H, dtype=torch.bool, device="cuda")
    ok[1, 5] = ok[0, 9] = False
    for g, c in zip(got[:5], clean[:5]):
        assert torch.equal(g[ok] if g.dim() == 2 else g[:, ok], c[ok] if c.dim() == 2 else c[:, ok])
    assert torch.equal(got[5][ok.all(0)], clean[5][ok.all(0)])


@pytest.mark.parametrize("T,E,H", [(5, 2, 70), (40, 3, 33), (700, 2, 70), (9000, 2, 70), (40, 3, 27500)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("gap", [1, 3])
def test_a_reset_hides_gates_that_are_no_numbers(hip, T, E, H, dtype, gap):
    """A gate that is no number some steps in front of a reset: its column from there up to the reset, forward, and from there back to the
    reset before, backward; everything else bit for bit."""
    r = T // 2
    a, normal = make(T, E, H, dtype, bias=True)
    a["resets"] = torch.zeros(T, E, dtype=torch.uint8, device="cuda")
    a["resets"][r] = 1
    a["resets"][0] = 1
    dy = normal(T, E, H).to(dtype)
    clean = hip.glr_forward(a["f"], a["x"], a["h0"], resets=a["resets"], bias=a["bias"], want_saved=True)
    gclean = hip.glr_backward(a["f"], a["x"], dy, clean[2], resets=a["resets"], bias=a["bias"])
    f, at = a["f"].clone(), max(r - gap, 0)
    f[at, 1, 5] = float("nan")
    y, last, saved = hip.glr_forward(f, a["x"], a["h0"], resets=a["resets"], bias=a["bias"], want_saved=True)
    df, dx, dh0, dbias = hip.glr_backward(f, a["x"], dy, saved, resets=a["resets"], bias=a["bias"])
    assert bool(torch.isnan(y[at:r, 1, 5]).all()) and bool(torch.isnan(df[:r, 1, 5]).any())
    rest = torch.ones_like(y, dtype=torch.bool)
    rest[at:r, 1, 5] = False
    assert torch.equal(y[rest], clean[0][rest]) and torch.equal(last, clean[1])
    rest[:r, 1, 5] = False
    assert torch.equal(df[rest], gclean[0][rest]) and torch.equal(dx[rest], gclean[1][rest]) and torch.equal(dh0, gclean[2])
    ok = torch.ones(H, dtype=torch.bool, device="cuda")
    ok[5] = False
    assert torch.equal(dbias[ok], gclean[3][ok]) and bool(torch.isnan(dbias[5]))
