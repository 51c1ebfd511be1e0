"""AdamW over many tensors on the GPU against its definition in 64 bits, moments in 32 and in 8 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
U = 2.0 ** -24
B1, B2 = 0.9, 0.999
BLOCK = 256


@pytest.fixture(scope="module")
def hip():
    from baselines_amd import hip
    return hip


LISTS = [[1], [3], [255, 1, 256, 257, 2], [2047, 2048, 2049], [17 * 64, 64, 64 * 64, 64, 64 * 6, 6, 6], [100003], [5, 0, 1030, 7], [4096 * 5 + 3, 9],
         [64] * 500]


def tensors(sizes, dtype, g, scale=1.0, odd=False):
    """Tensors of the sizes; `odd` packs them into one arena, so that they begin at any element."""
    if odd:
        flat = (scale * torch.randn(sum(sizes) + 1, generator=g, device="cuda")).to(dtype)
        got, at = [], 1
        for n in sizes:
            got.append(flat[at:at + n])
            at += n
        return got
    return [(scale * torch.randn(n, generator=g, device="cuda")).to(dtype) for n in sizes]


def reference(p, grads, m, v, lr, t, decay, wd=0.01, eps=1e-8, clip=0.0, gscale=1.0):
    """One step in 64 bits over packed lists; tensors whose gradient is None stay as they are."""
    live = [g is not None for g in grads]
    gs = [None if g is None else g.double() * gscale for g in grads]
    norm = sum(float(g.square().sum()) for g in gs if g is not None) ** 0.5
    factor = min(1.0, clip / norm) if clip > 0 and norm > 0 else 1.0
    out = []
    for k, on in enumerate(live):
        if not on:
            out.append((p[k], m[k], v[k], None))
            continue
        g = gs[k] * factor
        m1, v1 = B1 * m[k] + (1 - B1) * g, B2 * v[k] + (1 - B2) * g * g
        step = (m1 / (1 - B1 ** t)) / ((v1 / (1 - B2 ** t)).sqrt() + eps)
        out.append((p[k] - lr * (step + wd * decay[k] * p[k]), m1, v1, g))
    return [list(x) for x in zip(*out)], norm, factor


def close(got, want, tol, what):
    err = (got.double() - want).abs()
    if got.dtype == BF16:
        tol = (tol + 2.0 ** -8 * want.abs()) * (1 + 2.0 ** -7)
    bad = ~(err <= tol)
    assert not bool(bad.any()), (what, float(err[bad].max()), int(bad.sum()))


def tol_p(p, new, lr, m, m1, v1, t, g):
    """The new parameter rounds once (U of it) and p's share once more; the update lr step is off by the relative errors of m
    (m's own rounding, which is U of its terms, not of their sum), of v and its root, of the quotient and of the two corrections:
    at most 16 U of |lr step| plus 3 U of lr times m's terms over the root, and lr U of the decay."""
    root = (v1 / (1 - B2 ** t)).sqrt() + 1e-30
    terms = (B1 * m.abs() + (1 - B1) * g.abs()) / (1 - B1 ** t)
    return 2 * U * (new.abs() + p.abs()) + lr * (16 * U * (m1.abs() / (1 - B1 ** t)) / root + 4 * U * terms / root) + 4 * lr * U * p.abs()


@pytest.mark.parametrize("sizes", LISTS, ids=lambda s: "x".join(map(str, s[:4])) + ("..%d" % len(s) if len(s) > 4 else ""))
@pytest.mark.parametrize("pt,gt", [(F32, F32), (BF16, BF16), (BF16, F32), (F32, BF16)])
@pytest.mark.parametrize("clip", [0.0, 0.5])
def test_32_bits(hip, sizes, pt, gt, clip):
    g = torch.Generator(device="cuda").manual_seed(len(sizes))
    odd = len(sizes) % 2 == 1
    ps = tensors(sizes, pt, g, 0.1, odd)
    decay = [k % 2 for k in range(len(sizes))]
    plan = hip.AdamWPlan(ps, decay=decay, grad_dtype=gt)
    lr = 1e-2
    for t in (1, 2, 3):
        grads = tensors(sizes, gt, g, 0.3, odd)
        if len(sizes) > 3 and t == 2:
            grads[1] = None
        old = [p.double() for p in ps]
        m, v = ([s.double() for s in x.split(sizes)] for x in (plan.m, plan.v))
        hip.adamw_step(plan, grads, lr, t, max_grad_norm=clip, grad_scale=0.5)
        (np_, nm, nv, gs), norm, factor = reference(old, grads, m, v, lr, t, decay, clip=clip, gscale=0.5)
        got_m, got_v = plan.m.split(sizes), plan.v.split(sizes)
        for k in range(len(sizes)):
            if grads[k] is None:
                assert torch.equal(ps[k].double(), old[k]) and torch.equal(got_m[k].double(), m[k]) and torch.equal(got_v[k].double(), v[k])
                continue
            # g: scaled and clipped, three roundings and the norm's own; squares twice that
            close(got_m[k], nm[k], 4 * U * (B1 * m[k].abs() + (1 - B1) * gs[k].abs()) + 6 * U * (1 - B1) * gs[k].abs(), ("m", k, t))
            close(got_v[k], nv[k], 16 * U * nv[k], ("v", k, t))
            close(ps[k], np_[k], tol_p(old[k], np_[k], lr, m[k], nm[k], nv[k], t, gs[k]) + lr * 12 * U * (gs[k].abs() / ((nv[k] / (1 - B2 ** t)).sqrt() + 1e-30)),
                  ("p", k, t))
        if clip:
            assert abs(float(plan.norm[0]) - norm) <= 4 * U * norm
        assert abs(float(plan.norm[1]) - 0.5 * factor) <= 8 * U * factor


def blocks(sizes):
    return [-(-n // BLOCK) * BLOCK for n in sizes]


def unpad(x, sizes):
    return [q[:n] for q, n in zip(x.split(blocks(sizes)), sizes)]


def decode(plan, sizes):
    """Values of the codes by the definition, in 64 bits."""
    m = plan.m.double() / 127
    m = m * m.abs() * plan.m_scale.double().repeat_interleave(BLOCK)
    v = (plan.v.double() / 255) ** 4 * plan.v_scale.double().repeat_interleave(BLOCK)
    return unpad(m, sizes), unpad(v, sizes)


def check_codes(plan, sizes, m, v, dm, dv):
    """Scales are the blocks' largest values, and every code is the nearest one: the root of a value that is off by a share d of
    itself (by dm, dv in all) moves the code's place by 127 d / 2 (255 d / 4), and the roots and the product round by 6 U more."""
    for x, d, codes, scale, top, root in ((m, dm, plan.m, plan.m_scale, 127, 2), (v, dv, plan.v, plan.v_scale, 255, 4)):
        pad = lambda z: torch.cat([torch.nn.functional.pad(q, (0, b - q.numel())) for q, b in zip(z, blocks(sizes))]).view(-1, BLOCK)      # noqa: E731
        x, d = pad(x), pad(d)
        want = x.abs().amax(1)
        assert bool(((scale.double() - want).abs() <= d.amax(1) + U * want).all())
        place = top * (x.abs() / scale.double().clamp(min=1e-300).unsqueeze(1)) ** (1 / root)
        slack = top * (d / x.abs().clamp(min=1e-300)).clamp(max=1.0) / root + (d.amax(1) / want.clamp(min=1e-300) + 8 * U).unsqueeze(1) * top
        c = codes.double().view(-1, BLOCK)
        off = (c.abs() - place).abs()
        ok = off <= 0.5 + slack
        if root == 4:
            ok |= (c == 1) & (place < 1)
            assert bool((c[x > 0] > 0).all()), "a v that is not zero has code 0"
        assert bool(ok.all()), (root, float((off - slack).max()))
        clear = (place > 0.5 + slack)
        assert torch.equal(torch.sign(c[clear]), torch.sign(x[clear]))
        assert bool((c[x == 0] == 0).all())


@pytest.mark.parametrize("sizes", LISTS, ids=lambda s: "x".join(map(str, s[:4])) + ("..%d" % len(s) if len(s) > 4 else ""))
@pytest.mark.parametrize("pt,gt", [(F32, F32), (BF16, BF16), (F32, BF16)])
@pytest.mark.parametrize("clip", [0.0, 0.5])
def test_8_bits(hip, sizes, pt, gt, clip):
    g = torch.Generator(device="cuda").manual_seed(len(sizes))
    odd = len(sizes) % 2 == 1
    ps = tensors(sizes, pt, g, 0.1, odd)
    decay = [k % 2 for k in range(len(sizes))]
    plan = hip.AdamWPlan(ps, state_bits=8, decay=decay, grad_dtype=gt)
    assert plan.m.dtype == torch.int8 and plan.v.dtype == torch.uint8
    lr = 1e-2
    for t in (1, 2, 3):
        grads = [x * torch.exp(2 * torch.randn(x.shape, generator=g, device="cuda")).to(gt) for x in tensors(sizes, gt, g, 0.3)]
        old = [p.double() for p in ps]
        m, v = decode(plan, sizes)
        vals = hip.adamw_state(plan), hip.adamw_state(plan, dtype=BF16)
        for got, want in zip(vals[0], (m, v)):
            close(got, torch.cat(want), 8 * U * torch.cat(want).abs(), "state")          # a quotient, two or three products, the scale
        for got, want in zip(vals[1], (m, v)):
            close(got, torch.cat(want), 8 * U * torch.cat(want).abs(), "state in bfloat16")
        hip.adamw_step(plan, grads, lr, t, max_grad_norm=clip, grad_scale=2.0)
        (np_, nm, nv, gs), norm, factor = reference(old, grads, m, v, lr, t, decay, clip=clip, gscale=2.0)
        dm = [16 * U * (B1 * a.abs() + (1 - B1) * b.abs()) for a, b in zip(m, gs)]
        dv = [28 * U * b for b in nv]
        check_codes(plan, sizes, nm, nv, dm, dv)
        for k in range(len(sizes)):
            root = (nv[k] / (1 - B2 ** t)).sqrt() + 1e-30
            close(ps[k], np_[k], tol_p(old[k], np_[k], lr, m[k], nm[k], nv[k], t, gs[k]) + 2 * lr * (dm[k] / (1 - B1 ** t) / root + 14 * U * nm[k].abs() / root),
                  ("p", k, t))


def test_8_bits_track_32_over_many_steps(hip):
    """The same noisy quadratic with moments in 32 and in 8 bits: parameters end within a tenth of the way they went."""
    g = torch.Generator(device="cuda").manual_seed(0)
    start = [torch.randn(n, generator=g, device="cuda") for n in (1000, 64, 257)]
    ends = []
    for bits in (32, 8):
        ps = [p.clone() for p in start]
        plan = hip.AdamWPlan(ps, state_bits=bits)
        h = torch.Generator(device="cuda").manual_seed(1)
        for t in range(1, 101):
            hip.adamw_step(plan, [p + 0.1 * torch.randn(p.shape, generator=h, device="cuda") for p in ps], 5e-3, t)
        ends.append(torch.cat(ps))
    way = (ends[0] - torch.cat(start)).norm()
    assert float((ends[1] - ends[0]).norm()) < 0.1 * float(way)


@pytest.mark.parametrize("bits", [32, 8])
def test_what_is_not_a_number_stays_where_it_is(hip, bits):
    """Without clipping an infinity or NaN spoils its own element, and in 8 bits the moments of its block from then on."""
    sizes = [600, 300]
    g = torch.Generator(device="cuda").manual_seed(4)
    start, grads = tensors(sizes, F32, g), tensors(sizes, F32, g)
    clean, dirty = [p.clone() for p in start], [p.clone() for p in start]
    pc, pd = hip.AdamWPlan(clean, state_bits=bits), hip.AdamWPlan(dirty, state_bits=bits)
    hip.adamw_step(pc, grads, 1e-2, 1)
    bad = [x.clone() for x in grads]
    bad[0][300], bad[1][299] = float("nan"), float("inf")
    hip.adamw_step(pd, bad, 1e-2, 1)
    for k, at in ((0, 300), (1, 299)):
        ok = torch.ones(sizes[k], dtype=torch.bool, device="cuda")
        ok[at] = False
        assert torch.equal(clean[k][ok], dirty[k][ok]) and not bool(torch.isfinite(dirty[k][at]))
    m = hip.adamw_state(pd)[0].split(sizes)
    if bits == 8:
        assert bool(torch.isnan(m[0][256:512]).all()) and bool(torch.isnan(m[1][256:]).all())
        assert bool(torch.isfinite(m[0][:256]).all()) and bool(torch.isfinite(m[0][512:]).all()) and bool(torch.isfinite(m[1][:256]).all())
    # with clipping the norm carries it everywhere, as the formula says for NaN; an infinite norm leaves zero gradients
    hip.adamw_step(pd, bad, 1e-2, 2, max_grad_norm=1.0)
    assert bool(torch.isnan(pd.norm).all()) and bool(torch.isnan(dirty[1]).all())
    inf = [x.clone() for x in grads]
    inf[0][5] = float("inf")
    before = clean[1].clone()
    hip.adamw_step(pc, inf, 0.0, 2, max_grad_norm=1.0)
    assert float(pc.norm[0]) == float("inf") and float(pc.norm[1]) == 0.0 and torch.equal(clean[1], before)


@pytest.mark.parametrize("bits", [32, 8])
def test_zero_gradients_and_zero_moments(hip, bits):
    ps = [torch.ones(300, device="cuda"), torch.ones(5, device="cuda")]
    plan = hip.AdamWPlan(ps, state_bits=bits, decay=[1, 0])
    hip.adamw_step(plan, [torch.zeros(300, device="cuda"), torch.zeros(5, device="cuda")], 0.1, 1, weight_decay=0.5, max_grad_norm=1.0)
    assert float(plan.norm[0]) == 0.0 and float(plan.norm[1]) == 1.0
    assert bool(((ps[0] - 0.95).abs() <= 2 * U).all()) and bool((ps[1] == 1).all())
    m, v = hip.adamw_state(plan)
    assert bool((m == 0).all()) and bool((v == 0).all())
    hip.adamw_step(plan, [None, None], 0.1, 2, max_grad_norm=1.0)
    assert bool((ps[1] == 1).all()) and float(plan.norm[0]) == 0.0


@pytest.mark.parametrize("bits", [32, 8])
def test_neighbours_of_a_view_stay(hip, bits):
    arena = torch.full((5000,), 7.0, device="cuda")
    ps = [arena[3:1003], arena[1004:1005], arena[2001:4998]]
    plan = hip.AdamWPlan(ps, state_bits=bits)
    hip.adamw_step(plan, [torch.ones_like(p) for p in ps], 0.1, 1)
    keep = torch.ones(5000, dtype=torch.bool, device="cuda")
    for a, b in ((3, 1003), (1004, 1005), (2001, 4998)):
        keep[a:b] = False
    assert bool((arena[keep] == 7).all()) and bool((arena[~keep] != 7).all())


def test_adopted_state_and_refusals(hip):
    p = torch.zeros(300, device="cuda")
    m, v = torch.ones(300, device="cuda"), torch.ones(300, device="cuda")
    plan = hip.AdamWPlan([p], state=(m, v))
    hip.adamw_step(plan, [torch.zeros(300, device="cuda")], 0.1, 1)
    assert plan.m is m and bool((m - 0.9).abs().max() < 1e-6)
    assert hip.adamw_state(plan) == (m, v)
    z = torch.zeros
    for state in ((m,), (m, v[:200]), (m.double(), v), (m, v, m, v)):
        with pytest.raises((ValueError, TypeError)):
            hip.AdamWPlan([p], state=state)
    codes = (z(512, dtype=torch.int8, device="cuda"), z(2, device="cuda"), z(512, dtype=torch.uint8, device="cuda"), z(2, device="cuda"))
    hip.AdamWPlan([p], state_bits=8, state=codes)
    with pytest.raises(ValueError, match="aligned"):
        hip.AdamWPlan([p], state_bits=8, state=(z(513, dtype=torch.int8, device="cuda")[1:],) + codes[1:])
    for grads, err in (([], ValueError), ([z(300, device="cuda")] * 2, ValueError), ([z(299, device="cuda")], ValueError),
                       ([z(300, device="cuda", dtype=BF16)], TypeError), ([z(300)], TypeError), ([z(600, device="cuda")[::2]], ValueError)):
        with pytest.raises(err):
            hip.adamw_step(plan, grads, 0.1, 1)
    from baselines_amd import _lib
    with pytest.raises(_lib.Ppo2HipError, match="t=0"):
        hip.adamw_step(plan, [z(300, device="cuda")], 0.1, 0)
    with pytest.raises(_lib.Ppo2HipError, match="beta1"):
        hip.adamw_step(plan, [z(300, device="cuda")], 0.1, 1, beta1=1.0)
    with pytest.raises(TypeError):
        hip.adamw_state(plan, dtype=BF16)
    plan.params[0].set_(z(300, device="cuda"))
    with pytest.raises(ValueError, match="moved"):
        hip.adamw_step(plan, [z(300, device="cuda")], 0.1, 1)


@pytest.mark.parametrize("bits", [32, 8])
def test_same_bits_every_time_on_any_stream(hip, bits):
    sizes = [100003, 17, 4096, 2049]
    g = torch.Generator(device="cuda").manual_seed(9)
    start, grads = tensors(sizes, F32, g), tensors(sizes, F32, g)
    runs = []
    torch.cuda.synchronize()
    for s in (None, torch.cuda.Stream(), torch.cuda.Stream()):
        with torch.cuda.stream(s):
            ps = [p.clone() for p in start]
            plan = hip.AdamWPlan(ps, state_bits=bits)
            for t in (1, 2, 3):
                hip.adamw_step(plan, grads, 1e-2, t, max_grad_norm=0.5)
            m, v = hip.adamw_state(plan)
        runs.append(ps + [m, v, plan.norm])
        torch.cuda.synchronize()
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], r))


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_and_replayed(hip, bits):
    """A captured step replayed with new gradients in the same tensors, eager work between, against eager steps.  (lr and t are the
    captured call's.)"""
    sizes = [5003, 17, 2049]
    g = torch.Generator(device="cuda").manual_seed(9)
    start, grads = tensors(sizes, F32, g), tensors(sizes, F32, g)
    pg, pe = [p.clone() for p in start], [p.clone() for p in start]
    plan_g, plan_e = hip.AdamWPlan(pg, state_bits=bits), hip.AdamWPlan(pe, state_bits=bits)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        hip.adamw_step(plan_g, grads, 1e-2, 7, max_grad_norm=0.5)
    for _ in range(4):
        for x in grads:
            x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        hip.adamw_step(plan_e, grads, 1e-2, 7, max_grad_norm=0.5)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(pg + [plan_g.m, plan_g.v, plan_g.norm], pe + [plan_e.m, plan_e.v, plan_e.norm]))


def test_more_tensors_than_one_launch_takes(hip):
    """1000 tensors of one clipped step: the norm spans the launches."""
    n = 1000
    g = torch.Generator(device="cuda").manual_seed(5)
    sizes = [1 + (k * 37) % 300 for k in range(n)]
    ps, grads = tensors(sizes, F32, g, 1.0, True), tensors(sizes, F32, g)
    old = [p.double() for p in ps]
    plan = hip.AdamWPlan(ps)
    hip.adamw_step(plan, grads, 1e-2, 1, max_grad_norm=1.0)
    zero = [torch.zeros_like(o) for o in old]
    (np_, nm, nv, gs), norm, _ = reference(old, grads, zero, zero, 1e-2, 1, [1.0] * n, clip=1.0)
    assert abs(float(plan.norm[0]) - norm) <= 4 * U * norm
    for k in range(n):
        close(ps[k], np_[k], tol_p(old[k], np_[k], 1e-2, zero[k], nm[k], nv[k], 1, gs[k]) + 1e-2 * 12 * U * 2, ("p", k))


class _TwoRanks:
    """Stands for a communicator of two ranks that bring the same gradients."""
    size = 2

    def __init__(self):
        self.checks = self.casts = 0

    def allreduce_sum_(self, t):
        return t.mul_(2)

    def bcast_(self, t, root=0):
        self.casts += 1
        return t

    def check_synced(self, theta):
        self.checks += 1


@pytest.mark.parametrize("pt", [F32, BF16])
def test_mpi_adamw(hip, pt):
    from baselines_amd.common.mpi_adam import MpiAdamW
    sizes = [64, 17, 300]
    g = torch.Generator(device="cuda").manual_seed(5)
    start = tensors(sizes, pt, g)
    one, two = [p.clone() for p in start], [p.clone() for p in start]
    comm = _TwoRanks()
    a = MpiAdamW(one, max_grad_norm=0.5, grad_dtype=F32)
    b = MpiAdamW(two, max_grad_norm=0.5, comm=comm)
    for _ in range(3):
        grads = tensors(sizes, F32, g)
        a.update(grads, 1e-2)
        b.update(grads, 1e-2)
    assert a.t == b.t == 3 and comm.checks == 1
    assert all(torch.equal(x, y) for x, y in zip(one, two))       # 2 g / 2 is g exactly
    b.sync()
    assert comm.casts == 3
    with pytest.raises(ValueError, match="every rank"):
        b.update([None] + grads[1:], 1e-2)
    a.update([None] + grads[1:], 1e-2)


def test_training_a_recurrent_layer(hip):
    """The operators as they are used: projection, recurrence forward and backward, AdamW, over three rollouts whose last states
    go on; parameters against the same in 64 bits with automatic gradients."""
    T, E, D, H, lr = 40, 6, 12, 32, 1e-2
    g = torch.Generator(device="cuda").manual_seed(11)
    w = torch.randn(D, 2 * H, generator=g, device="cuda") / D ** 0.5
    bias, head = 2 * torch.rand(H, generator=g, device="cuda"), torch.randn(H, 1, generator=g, device="cuda") / H ** 0.5
    wide = [p.double().requires_grad_() for p in (w, bias, head)]
    ref_m, ref_v = ([torch.zeros_like(p) for p in wide] for _ in range(2))
    plan = hip.AdamWPlan([w, bias, head], decay=[1, 0, 1])
    state, wstate = torch.zeros(E, H, device="cuda"), torch.zeros(E, H, dtype=torch.float64, device="cuda")
    for t in range(1, 4):
        obs = torch.randn(T, E, D, generator=g, device="cuda")
        target = torch.randn(T, E, 1, generator=g, device="cuda")
        dones = torch.rand(T, E, generator=g, device="cuda") < 0.1
        joint = obs.view(T * E, D).mm(w).view(T, E, 2 * H)
        y, state, saved = hip.glr_forward(joint[..., :H], joint[..., H:], state, resets=dones, bias=bias, want_saved=True)
        err = y.view(T * E, H).mm(head) - target.view(T * E, 1)
        dout = err * (2.0 / (T * E))
        dhead = y.view(T * E, H).t().contiguous().mm(dout)
        dy = dout.mm(head.t().contiguous()).view(T, E, H)
        djoint = torch.empty_like(joint)
        _, _, _, dbias = hip.glr_backward(joint[..., :H], joint[..., H:], dy, saved, resets=dones, bias=bias, df=djoint[..., :H], dx=djoint[..., H:])
        dw = obs.view(T * E, D).t().contiguous().mm(djoint.view(T * E, 2 * H))
        hip.adamw_step(plan, [dw, dbias, dhead], lr, t, max_grad_norm=1.0)

        wj = obs.double().view(T * E, D).mm(wide[0]).view(T, E, 2 * H)
        h, ys = wstate, []
        for s in range(T):
            a = torch.sigmoid(wj[s, :, :H] + wide[1])
            h = a * torch.where(dones[s].unsqueeze(-1), 0.0, h) + (1 - a) * wj[s, :, H:]
            ys.append(h)
        wstate = h.detach()
        loss = (torch.stack(ys).view(T * E, H).mm(wide[2]) - target.double().view(T * E, 1)).square().mean()
        grads = torch.autograd.grad(loss, wide)
        for got, want in zip((dw, dbias, dhead), grads):
            assert float((got.double() - want).norm() / want.norm()) < 1e-4
        (new, ref_m, ref_v, _), _, _ = reference([p.detach() for p in wide], list(grads), ref_m, ref_v, lr, t, [1, 0, 1], clip=1.0)
        wide = [p.requires_grad_() for p in new]
    # Adam divides by the root of v: an element whose gradient is far below its tensor's norm may step any way within lr
    for got, want in zip((w, bias, head), wide):
        assert float((got.double() - want.detach()).norm() / want.detach().norm()) < 1e-3


@pytest.mark.parametrize("sizes", [[700, 3], [40000]])
@pytest.mark.parametrize("eps", [0.0, 1e-38, 1e-30, 1e-12, 1e-8, 1.0])
@pytest.mark.parametrize("scale", [1e-15, 1.0])
def test_small_and_large_epsilons(hip, sizes, eps, scale):
    """Gradients whose squares are near the smallest normal numbers, with an epsilon on either side of their roots."""
    g = torch.Generator(device="cuda").manual_seed(7)
    ps = tensors(sizes, F32, g, 0.1)
    plan = hip.AdamWPlan(ps)
    lr = 1e-2
    for t in (1, 2):
        grads = [scale * torch.sign(x) * (0.5 + torch.rand(x.shape, generator=g, device="cuda")) for x in tensors(sizes, F32, g)]
        old = [p.double() for p in ps]
        m, v = ([s.double() for s in x.split(sizes)] for x in (plan.m, plan.v))
        hip.adamw_step(plan, grads, lr, t, epsilon=eps, weight_decay=0.0, max_grad_norm=1e30)
        (new, nm, nv, gs), _, _ = reference(old, grads, m, v, lr, t, [0] * len(sizes), wd=0.0, eps=eps)
        for k in range(len(sizes)):
            close(ps[k], new[k], tol_p(old[k], new[k], lr, m[k], nm[k], nv[k], t, gs[k]), ("p", k, t))


def test_what_a_plan_refuses_to_share(hip):
    """Moments in one place with each other or with a parameter, a parameter whose storage was exchanged behind the plan, and gradients
    that are no tensors."""
    z = lambda n, dt=F32: torch.zeros(n, dtype=dt, device="cuda")      # noqa: E731
    p, both = z(300), z(700)
    for state in ((both[:300], both[200:500]), (both[:300], both[:300]), (p, z(300))):
        with pytest.raises(ValueError, match="overlaps"):
            hip.AdamWPlan([p], state=state)
    plan = hip.AdamWPlan([p], state=(both[:300], both[300:600]))
    with pytest.raises(TypeError):
        hip.adamw_step(plan, [3.0], 0.1, 1)
    layer = torch.nn.Linear(3, 2, device="cuda")
    plan = hip.AdamWPlan(layer.parameters())
    grads = [torch.ones_like(q) for q in plan.params]
    hip.adamw_step(plan, grads, 0.1, 1)
    layer.weight.data = layer.weight.data.clone()
    with pytest.raises(ValueError, match="moved"):
        hip.adamw_step(plan, grads, 0.1, 2)


@pytest.mark.parametrize("bits", [32, 8])
def test_moments_that_were_exchanged_are_refused(hip, bits):
    """A plan holds its arrays' addresses: a step after one of them was replaced would go on in the old one."""
    p, grads = [torch.ones(300, device="cuda")], [torch.ones(300, device="cuda")]
    names = ["m", "v", "norm"] + (["m_scale", "v_scale"] if bits == 8 else [])
    for name in names:
        for how in ("attribute", "data"):
            plan = hip.AdamWPlan(p, state_bits=bits)
            hip.adamw_step(plan, grads, 0.1, 1)
            old = getattr(plan, name)
            before = old.clone(), p[0].clone()
            if how == "attribute":
                setattr(plan, name, old.clone())
            else:
                keep = old.data         # what the plan still points at stays allocated
                old.data = old.clone()
            with pytest.raises(ValueError, match="moved"):
                hip.adamw_step(plan, grads, 0.1, 2)
            assert torch.equal(p[0], before[1])
            if name != "norm" and bits == 8:
                with pytest.raises(ValueError, match="moved"):
                    hip.adamw_state(plan)
            if how == "attribute":
                assert torch.equal(old, before[0])
                setattr(plan, name, old)
                hip.adamw_step(plan, grads, 0.1, 2)
    # new values in the same memory are what a plan takes
    plan = hip.AdamWPlan(p, state_bits=bits)
    plan.m.copy_(torch.ones_like(plan.m))
    hip.adamw_step(plan, grads, 0.1, 1)


def test_gradients_have_their_tensors_shapes(hip):
    """An [H, D] gradient has as many entries as its [D, H] tensor, and none of them in its place.  Dimensions of one and flat
    gradients change no order."""
    p = [torch.ones(4, 6, device="cuda"), torch.ones(5, device="cuda"), torch.ones((), device="cuda")]
    plan = hip.AdamWPlan(p)
    z = lambda *s: torch.ones(s, device="cuda")      # noqa: E731
    for k, bad in ((0, z(6, 4)), (0, z(2, 12)), (0, z(4, 3, 2)), (1, z(6)), (1, z(5, 2)), (2, z(2))):
        grads = [z(4, 6), z(5), z()]
        grads[k] = bad
        before = [q.clone() for q in p]
        with pytest.raises(ValueError, match=r"grads\[%d\]" % k):
            hip.adamw_step(plan, grads, 0.1, 1)
        assert all(torch.equal(a, b) for a, b in zip(p, before))
    for t, grads in enumerate(([z(4, 6), z(5), z()], [z(24), z(5, 1), z(1)], [z(1, 4, 6), None, z(1, 1)]), 1):
        hip.adamw_step(plan, grads, 0.1, t)
    one = z(4, 6)                                   # the same tensor twice: right for the first, wrong for the second
    plan = hip.AdamWPlan([z(4, 6), z(6, 4)])
    with pytest.raises(ValueError, match=r"grads\[1\]"):
        hip.adamw_step(plan, [one, one], 0.1, 1)
    hip.adamw_step(plan, [one, one.view(6, 4)], 0.1, 1)


def test_mpi_adamw_gradients_of_wrong_shapes(hip):
    """With several ranks as in a single process: nothing is broadcast into a tensor's gradient."""
    from baselines_amd.common.mpi_adam import MpiAdamW
    p = [torch.ones(4, 6, device="cuda"), torch.ones(5, device="cuda")]
    a, b = [q.clone() for q in p], [q.clone() for q in p]
    one, two = MpiAdamW(a), MpiAdamW(b, comm=_TwoRanks())
    z = lambda *s: torch.rand(s, device="cuda")      # noqa: E731
    for k, bad in ((0, z(6)), (0, z(1)), (0, z(6, 4)), (0, z(4, 1)), (1, z(1)), (1, z())):
        grads = [z(4, 6), z(5)]
        grads[k] = bad
        for opt in (one, two):
            with pytest.raises(ValueError, match=r"grads\[%d\]" % k):
                opt.update(grads, 0.1)
        assert one.t == two.t == 0
    for grads in ([z(4, 6), z(5)], [z(24), z(5, 1)]):
        one.update(grads, 0.1)
        two.update(grads, 0.1)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_mpi_adamw_goes_on_from_adopted_state(hip):
    """Three steps, and two more by a second object that takes the first one's moments and its count: five steps in a row."""
    from baselines_amd.common.mpi_adam import MpiAdamW
    g = torch.Generator(device="cuda").manual_seed(3)
    start = tensors([64, 300], F32, g)
    grads = [tensors([64, 300], F32, g) for _ in range(5)]
    one, two = [p.clone() for p in start], [p.clone() for p in start]
    a, b = MpiAdamW(one), MpiAdamW(two)
    for k in range(5):
        a.update(grads[k], 1e-2)
    for k in range(3):
        b.update(grads[k], 1e-2)
    c = MpiAdamW(two, state=(b.plan.m, b.plan.v), t=b.t)
    for k in (3, 4):
        c.update(grads[k], 1e-2)
    assert c.t == 5
    assert all(torch.equal(p, q) for p, q in zip(one, two)) and torch.equal(a.plan.m, c.plan.m) and torch.equal(a.plan.v, c.plan.v)
    for t in (-1, 1.5, None):
        with pytest.raises((ValueError, TypeError)):
            MpiAdamW(two, t=t)


# chunks of 2048 elements: 601 (a norm whose workgroups take more than one, its sums added up by every workgroup of the step), 2101
# (more sums than those add up: a launch of its own finds norm and factor), and both over lists of more than one launch's tensors
WIDE = [[600 * 2048 + 5], [2100 * 2048 + 7], [3, 2049 * 2048, 1], [5 * 2048 - 3] * 500, [700] * 1000 + [1500 * 2048 + 1]]


@pytest.mark.parametrize("sizes", WIDE, ids=lambda s: "%dx%d" % (len(s), max(s)))
@pytest.mark.parametrize("pt", [F32, BF16])
@pytest.mark.parametrize("clip", [0.0, 0.5])
def test_wide_lists_32_bits(hip, sizes, pt, clip):
    test_32_bits(hip, sizes, pt, F32, clip)


@pytest.mark.parametrize("sizes", WIDE, ids=lambda s: "%dx%d" % (len(s), max(s)))
@pytest.mark.parametrize("clip", [0.0, 0.5, 1e9])
def test_wide_lists_8_bits(hip, sizes, clip):
    test_8_bits(hip, sizes, F32, F32, clip)
    g = torch.Generator(device="cuda").manual_seed(1)
    plan = hip.AdamWPlan(tensors(sizes, F32, g, 0.1), state_bits=8)
    grads = tensors(sizes, F32, g, 0.3)
    for t, none in enumerate((None, len(sizes) // 2), 1):
        if none is not None:
            grads[none] = None
        before = [p.clone() for p in plan.params], plan.m.clone()
        hip.adamw_step(plan, grads, 0.1, t, max_grad_norm=clip, grad_scale=2.0)
        norm = sum(float(x.double().square().sum()) for x in grads if x is not None) ** 0.5 * 2.0
        factor = min(1.0, clip / norm) if clip and norm else 1.0
        if clip:
            assert abs(float(plan.norm[0]) - norm) <= 4 * U * norm
        assert abs(float(plan.norm[1]) - 2.0 * factor) <= 16 * U * factor
        for k in range(len(sizes)):
            if k == none:
                assert torch.equal(plan.params[k], before[0][k])
        if none is not None:
            assert torch.equal(unpad(plan.m, sizes)[none], unpad(before[1], sizes)[none])


@pytest.mark.parametrize("bits", [32, 8])
def test_wide_lists_captured_and_replayed(hip, bits):
    """The three launches of a wide clipped list in a graph, replayed with new gradients, against eager steps."""
    sizes = [2100 * 2048 + 7, 300]
    g = torch.Generator(device="cuda").manual_seed(9)
    start, grads = tensors(sizes, F32, g), tensors(sizes, F32, g)
    pg, pe = [p.clone() for p in start], [p.clone() for p in start]
    plan_g, plan_e = hip.AdamWPlan(pg, state_bits=bits), hip.AdamWPlan(pe, state_bits=bits)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        hip.adamw_step(plan_g, grads, 1e-2, 7, max_grad_norm=0.5)
    for _ in range(4):
        for x in grads:
            x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        hip.adamw_step(plan_e, grads, 1e-2, 7, max_grad_norm=0.5)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(pg + [plan_g.m, plan_g.v, plan_g.norm], pe + [plan_e.m, plan_e.v, plan_e.norm]))
