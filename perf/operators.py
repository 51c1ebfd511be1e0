"""Cases that time the gated linear recurrence and the AdamW step over many tensors, with both in plain torch operations.

``own`` False computes a case from its formulas with elementary torch operations, ``own`` True through
``baselines_amd.hip``.

Recurrence, f and x [T, E, H]:   a = sigmoid(f + bias)    h_t = a_t p_t + (1 - a_t) x_t,   p_t = 0 where resets[t], else h_{t-1}
AdamW, moments m and v:          p -= lr (m / (1 - beta1^t) / (sqrt(v / (1 - beta2^t)) + eps) + weight_decay decay p)
8-bit moments, per block of 256 elements of one tensor:  m = s sign(c) (c / 127)^2,  v = s (c / 255)^4
"""
import math

import torch

own = False

BLOCK = 256
BETA1, BETA2, EPS, DECAY, LR, MAX_NORM = 0.9, 0.999, 1e-8, 0.01, 3e-4, 0.5
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


# ------------------------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------------------------

def _glr(name, op, T, E, H, dtype, resets=False, bias=False, layout="apart"):
    return dict(name=name, op=op, T=T, E=E, H=H, dtype=dtype, resets=resets, bias=bias, layout=layout)


def _adamw(name, net, width, depth, bits, dtype="f32", clip=True):
    return dict(name=name, op="adamw", net=net, width=width, depth=depth, bits=bits, dtype=dtype, clip=clip)


def listed():
    return [
        # one acting step of a rollout: the state of every env advances by one observation
        _glr("step e2048 h256 f32", "step", 1, 2048, 256, "f32", resets=True),
        # acting for few envs, gate and input straight from one projection, a width that no vector divides
        _glr("step e37 h333 bf16", "step", 1, 37, 333, "bf16", bias=True, layout="joint"),
        # a rollout's pass over the recurrent layer, with the dones of its envs
        _glr("forward t128 e512 h256 bf16", "forward", 128, 512, 256, "bf16", resets=True, bias=True),
        # one long sequence: the time axis has to be split to fill the card
        _glr("forward t65536 e1 h1000 bf16", "forward", 65536, 1, 1000, "bf16", bias=True, layout="joint"),
        # ragged sizes, evaluation of few envs
        _glr("forward t1001 e7 h333 f32", "forward", 1001, 7, 333, "f32", resets=True, layout="batch first"),
        # training on a rollout: forward, then the gradients of gate, input, bias and first state
        _glr("train t128 e512 h256 f32", "train", 128, 512, 256, "f32", resets=True, bias=True),
        # training on long sequences, joint projection
        _glr("train t16384 e4 h1024 bf16", "train", 16384, 4, 1024, "bf16", bias=True, layout="joint"),
        # the 13 tensors of the 64-64 actor and value trunks: latency
        _adamw("adamw mlp 64 f32", "mlp", 64, 2, 32),
        # a stack of wide layers, every tensor float32
        _adamw("adamw stack 1024x10 f32", "stack", 1024, 10, 32),
        # parameters and gradients in bfloat16, odd widths, no clipping
        _adamw("adamw stack 777x6 bf16", "stack", 777, 6, 32, "bf16", clip=False),
        # the convolutional policy with its recurrent layer, moments in 8 bits
        _adamw("adamw8 cnn 256 f32", "cnn", 256, 1, 8),
        # the wide stack, moments in 8 bits
        _adamw("adamw8 stack 1024x10 f32", "stack", 1024, 10, 8),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["step", "forward", "train", "adamw", "adamw"])
    if op == "adamw":
        net = rng.choice(["mlp", "cnn", "stack"])
        width = {"mlp": lambda: _log(rng, 16, 512), "cnn": lambda: _log(rng, 32, 512), "stack": lambda: _log(rng, 96, 1024)}[net]()
        depth = {"mlp": lambda: rng.randint(1, 4), "cnn": lambda: 1, "stack": lambda: _log(rng, 1, 10)}[net]()
        c = _adamw("", net, width, depth, rng.choice([8, 32]), rng.choice(["f32", "f32", "bf16"]), rng.random() < 0.6)
    else:
        H = _log(rng, 8, 2048)
        E = _log(rng, 1, 4096)
        T = 1 if op == "step" else _log(rng, 1, max(1, min(65536, (1 << 26) // (E * H))))
        c = _glr("", op, T, E, H, rng.choice(["f32", "bf16", "f16"]), rng.random() < 0.5, rng.random() < 0.5,
                 rng.choice(["apart", "joint", "batch first"]))
    del c["name"]
    return c


def work(case):
    if case["op"] == "adamw":
        n = sum(math.prod(s) for s in _shapes(case))
        es = SIZE[case["dtype"]]
        per = 3 * es + (16 if case["bits"] == 32 else 4 + 16 / BLOCK + 4)      # 8 bits: the moments are also handed out in 16
        return {"bytes": n * per, "flops": n * (16 if case["clip"] else 14)}
    es, EH = SIZE[case["dtype"]], case["E"] * case["H"]
    n = case["T"] * EH
    small = 8 * EH + (4 * case["H"] if case["bias"] else 0) + (case["T"] * case["E"] if case["resets"] else 0)
    if case["op"] == "train":
        return {"bytes": 6 * n * es + small + 8 * EH + (4 * case["H"] if case["bias"] else 0), "flops": 30 * n}
    return {"bytes": 3 * n * es + small, "flops": 10 * n}


# ------------------------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------------------------

def _shapes(case):
    """Shapes of a network's tensors in the order in which they are made."""
    w, d = case["width"], case["depth"]
    if case["net"] == "mlp":                       # two trunks of tanh layers, 17 observations, 6 actions
        trunk = [s for k in range(d) for s in ((17 if k == 0 else w, w), (w,))]
        return trunk + trunk + [(w, 6), (6,), (6,), (w, 1), (1,)]
    if case["net"] == "cnn":                       # three convolutions, a dense layer, a recurrent one of width w, two heads
        return [(8, 8, 4, 32), (32,), (4, 4, 32, 64), (64,), (3, 3, 64, 64), (64,), (3136, 512), (512,), (512, 4 * w), (w, 4 * w),
                (4 * w,), (w, 6), (6,), (w, 1), (1,)]
    return [s for _ in range(d) for s in ((w,), (w, w), (w, w), (w, w), (w, w), (w,), (w, 4 * w), (4 * w,), (4 * w, w), (w,))]


def _views(flat, shapes):
    got, at = [], 0
    for s in shapes:
        n = math.prod(s)
        got.append(flat[at:at + n].view(s))
        at += n
    return got


def _places(shapes):
    """Where every element of the packed list stands among blocks that begin anew with every tensor, and their number."""
    got, at = [], 0
    for s in shapes:
        n = math.prod(s)
        got.append(torch.arange(at, at + n, device="cuda"))
        at += -(-n // BLOCK) * BLOCK
    return torch.cat(got), at


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "adamw":
        return _prepare_adamw(case, g)
    T, E, H, dt = case["T"], case["E"], case["H"], TYPES[case["dtype"]]
    normal = lambda *s: torch.randn(s, generator=g, device="cuda")      # noqa: E731
    reach = 8 * torch.rand(H, generator=g, device="cuda")               # memories of one step to a few thousand
    s = {"op": case["op"], "T": T, "bias": reach if case["bias"] else None, "state": normal(E, H), "layout": case["layout"]}
    gate = normal(T, E, H) if case["bias"] else normal(T, E, H) + reach
    if case["layout"] == "joint":
        joint = torch.empty((T, E, 2 * H), dtype=dt, device="cuda")
        s["f"], s["x"] = joint[..., :H], joint[..., H:]
    elif case["layout"] == "batch first":
        s["f"], s["x"] = (torch.empty((E, T, H), dtype=dt, device="cuda").transpose(0, 1) for _ in range(2))
    else:
        s["f"], s["x"] = (torch.empty((T, E, H), dtype=dt, device="cuda") for _ in range(2))
    s["f"].copy_(gate)
    s["x"].copy_(normal(T, E, H))
    s["resets"] = torch.rand((T, E), generator=g, device="cuda") < 1 / 64 if case["resets"] else None
    if case["op"] == "train":
        s["dy"] = normal(T, E, H).to(dt)
        s["dh_last"] = normal(E, H)
    return s


def _prepare_adamw(case, g):
    shapes, dt = _shapes(case), TYPES[case["dtype"]]
    n = sum(math.prod(s) for s in shapes)
    s = {"op": "adamw", "bits": case["bits"], "t": 1000, "clip": MAX_NORM if case["clip"] else 0.0}
    normal = lambda: torch.randn(n, generator=g, device="cuda")         # noqa: E731
    spread = torch.exp(1.5 * normal())                                  # gradients of elements differ in size
    s["p"], s["g"] = (0.05 * normal()).to(dt), (1e-3 * spread * normal()).to(dt)
    m, v = 3e-4 * spread * normal(), 1e-6 * spread.square() * (0.5 + torch.rand(n, generator=g, device="cuda"))
    decays = [len(x) > 1 for x in shapes]
    if case["bits"] == 8:
        pos, npad = _places(shapes)
        s["state"] = _encode(m, v, pos, npad)
    else:
        s["state"] = (m, v)
    if own:
        from baselines_amd import hip
        s["grads"] = _views(s["g"], shapes)
        s["plan"] = hip.AdamWPlan(_views(s["p"], shapes), state_bits=case["bits"], decay=decays, state=s["state"])
    else:
        s["decay"] = torch.cat([torch.full((math.prod(x),), float(d), device="cuda") for x, d in zip(shapes, decays)])
        if case["bits"] == 8:
            s["pos"], s["npad"] = pos, npad
    return s


# ------------------------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------------------------

def run(s):
    if s["op"] == "adamw":
        s["t"] += 1
        return _adamw_own(s) if own else _adamw_plain(s)
    return _glr_own(s) if own else _glr_plain(s)


def _glr_own(s):
    from baselines_amd import hip
    if s["op"] == "step":
        y = hip.glr_step(s["f"][0], s["x"][0], s["state"], resets=None if s["resets"] is None else s["resets"][0], bias=s["bias"])
        return {"y": y, "state": s["state"]}
    train = s["op"] == "train"
    y, h_last, saved = hip.glr_forward(s["f"], s["x"], s["state"], resets=s["resets"], bias=s["bias"], want_saved=train)
    out = {"y": y, "h_last": h_last}
    if train:
        joint = None
        if s["layout"] == "joint":
            joint = torch.empty(s["f"].shape[:2] + (2 * s["f"].shape[2],), dtype=s["f"].dtype, device="cuda")
        H = s["f"].shape[2]
        df, dx, dh0, dbias = hip.glr_backward(s["f"], s["x"], s["dy"], saved, resets=s["resets"], bias=s["bias"], dh_last=s["dh_last"],
                                              df=None if joint is None else joint[..., :H], dx=None if joint is None else joint[..., H:])
        out.update({"df": df, "dx": dx, "dh0": dh0, "dbias": dbias} if joint is None else {"dfx": joint, "dh0": dh0, "dbias": dbias})
    return out


def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t from h_{-1} = 0 and the products of a, by joining spans of 1, 2, 4, ... steps."""
    d = 1
    while d < a.shape[0]:
        b = torch.cat([b[:d], b[d:] + a[d:] * b[:-d]])
        a = torch.cat([a[:d], a[d:] * a[:-d]])
        d *= 2
    return a, b


def _glr_plain(s):
    # 64 bits: products of thousands of gates next to one, and sums over all steps
    dt, x = s["x"].dtype, s["x"].double()
    z = s["f"].double() if s["bias"] is None else s["f"].double() + s["bias"]
    a, om = torch.sigmoid(z), torch.sigmoid(-z)
    through = a if s["resets"] is None else a * (~s["resets"]).unsqueeze(-1)
    grown, h = _scan(through, om * x)
    h = h + grown * s["state"]
    if s["op"] == "step":
        s["state"].copy_(h[-1])
        return {"y": h[-1].to(dt), "state": s["state"]}
    out = {"y": h.to(dt), "h_last": h[-1].float()}
    if s["op"] == "train":
        before = torch.cat([s["state"].double().unsqueeze(0), h[:-1]])
        if s["resets"] is not None:
            before = before * (~s["resets"]).unsqueeze(-1)
        dy = s["dy"].double()
        dy[-1] += s["dh_last"]
        after = torch.cat([through[1:], torch.zeros_like(through[:1])])
        g = _scan(after.flip(0), dy.flip(0))[1].flip(0)
        df, dx = g * (before - x) * a * om, om * g
        dh0 = (through[0] * g[0]).float()
        dbias = None if s["bias"] is None else df.sum((0, 1)).float()
        if s["layout"] == "joint":
            out.update(dfx=torch.cat([df, dx], -1).to(dt), dh0=dh0, dbias=dbias)
        else:
            out.update(df=df.to(dt), dx=dx.to(dt), dh0=dh0, dbias=dbias)
    return out


def _adamw_own(s):
    from baselines_amd import hip
    hip.adamw_step(s["plan"], s["grads"], LR, s["t"], beta1=BETA1, beta2=BETA2, epsilon=EPS, weight_decay=DECAY, max_grad_norm=s["clip"])
    m, v = s["state"] if s["bits"] == 32 else hip.adamw_state(s["plan"], dtype=torch.bfloat16)
    return {"p": s["p"], "m": m, "v": v}


def _decode(state, pos):
    mc, ms, vc, vs = state
    m, v = mc.float() / 127, vc.float() / 255
    m = (m * m.abs()).view(-1, BLOCK) * ms.unsqueeze(1)
    v = v.square().square().view(-1, BLOCK) * vs.unsqueeze(1)
    return m.view(-1)[pos], v.view(-1)[pos]


def _encode(m, v, pos, npad):
    mp, vp = (torch.zeros(npad, device="cuda").index_copy_(0, pos, x).view(-1, BLOCK) for x in (m, v))
    ms, vs = mp.abs().amax(1), vp.amax(1)
    mc = torch.round(mp.abs().sqrt() * torch.where(ms > 0, 127 / ms.sqrt(), 0.0).unsqueeze(1)) * mp.sign()
    vc = torch.round(vp.sqrt().sqrt() * torch.where(vs > 0, 255 / vs.sqrt().sqrt(), 0.0).unsqueeze(1))
    vc = torch.maximum(vc, (vp > 0).float())
    return mc.view(-1).to(torch.int8), ms, vc.view(-1).to(torch.uint8), vs


def _adamw_plain(s):
    p, g = s["p"].float(), s["g"].float()
    m, v = s["state"] if s["bits"] == 32 else _decode(s["state"], s["pos"])
    if s["clip"]:
        norm = torch.sqrt((g * g).sum(dtype=torch.float64)).float()
        g = g * (s["clip"] / torch.clamp(norm, min=s["clip"]))
    m, v = m * BETA1 + g * (1 - BETA1), v * BETA2 + g * g * (1 - BETA2)
    step = m * (1 / (1 - BETA1 ** s["t"])) / (torch.sqrt(v * (1 / (1 - BETA2 ** s["t"]))) + EPS)
    s["p"].copy_(p - LR * (step + p * (DECAY * s["decay"])))
    if s["bits"] == 32:
        s["state"][0].copy_(m)
        s["state"][1].copy_(v)
        return {"p": s["p"], "m": s["state"][0], "v": s["state"][1]}
    s["state"] = _encode(m, v, s["pos"], s["npad"])
    m, v = _decode(s["state"], s["pos"])
    return {"p": s["p"], "m": m.bfloat16(), "v": v.bfloat16()}


# ------------------------------------------------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# ------------------------------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return _exact_adamw(case, s) if case["op"] == "adamw" else _exact_glr(case, s)


def _exact_glr(case, s):
    T, f, x = case["T"], s["f"].to(torch.float64), s["x"].to(torch.float64)
    if s["bias"] is not None:
        f = f + s["bias"].to(torch.float64)
    keep = 1 / (1 + torch.exp(-f))
    take = 1 / (1 + torch.exp(f))
    del f
    zero = torch.zeros(1, 1, dtype=torch.float64, device="cuda")
    cut = None if s["resets"] is None else s["resets"].unsqueeze(-1)
    h, before, state = torch.empty_like(x), torch.empty_like(x), s["state"].to(torch.float64)
    fresh = take * x
    for t in range(T):
        before[t] = state if cut is None else torch.where(cut[t], zero, state)
        torch.addcmul(fresh[t], keep[t], before[t], out=h[t])
        state = h[t]
    if case["op"] == "step":
        return {"y": h[0], "state": h[0]}
    out = {"y": h, "h_last": h[T - 1]}
    if case["op"] == "train":
        g = s["dy"].to(torch.float64)
        back = s["dh_last"].to(torch.float64)
        for t in range(T - 1, -1, -1):
            g[t] += back
            back = keep[t] * g[t]
            if cut is not None:
                back = torch.where(cut[t], zero, back)
        df = (before - x) * keep * take * g
        dx = take * g
        dbias = None if s["bias"] is None else df.sum(dim=0).sum(dim=0)
        if s["layout"] == "joint":
            out.update(dfx=torch.cat([df, dx], dim=2), dh0=back, dbias=dbias)
        else:
            out.update(df=df, dx=dx, dh0=back, dbias=dbias)
    return out


def _exact_adamw(case, s):
    shapes = _shapes(case)
    p, g = s["p"].to(torch.float64), s["g"].to(torch.float64)
    pads = [-(-math.prod(x) // BLOCK) * BLOCK for x in shapes]
    if case["bits"] == 8:
        mc, ms, vc, vs = (x.to(torch.float64) for x in s["state"])
        m = torch.sign(mc) * torch.pow(mc / 127, 2) * ms.repeat_interleave(BLOCK)
        v = torch.pow(vc / 255, 4) * vs.repeat_interleave(BLOCK)
        unpad = lambda a: torch.cat([q[:math.prod(x)] for q, x in zip(a.split(pads), shapes)])      # noqa: E731
        m, v = unpad(m), unpad(v)
    else:
        m, v = (x.to(torch.float64) for x in s["state"])
    t = s["t"] + 1
    if s["clip"]:
        norm = math.sqrt(float(torch.dot(g, g)))
        if norm > s["clip"]:
            g = g * s["clip"] / norm
    m = m + (g - m) * (1 - BETA1)
    v = v + (g * g - v) * (1 - BETA2)
    new = []
    for q, d, x in zip(p.split([math.prod(x) for x in shapes]),
                       (m / (1 - math.pow(BETA1, t)) / ((v / (1 - math.pow(BETA2, t))).sqrt() + EPS)).split([math.prod(x) for x in shapes]), shapes):
        new.append(q * (1 - LR * DECAY) - LR * d if len(x) > 1 else q - LR * d)
    if case["bits"] == 8:
        def held(a, top, root):
            padded = torch.cat([torch.nn.functional.pad(q, (0, k - q.numel())) for q, k in zip(a.split([math.prod(x) for x in shapes]), pads)])
            size = padded.abs().view(-1, BLOCK)
            scale = size.max(dim=1, keepdim=True).values
            code = torch.round(top * torch.pow(size / torch.where(scale > 0, scale, 1.0), 1 / root))
            code = torch.where((code == 0) & (size > 0) & (root == 4), 1.0, code)
            return unpad((torch.pow(code / top, root) * scale).view(-1) * torch.sign(padded))
        m, v = held(m, 127, 2), held(v, 255, 4)
    return {"p": torch.cat(new), "m": m, "v": v}
