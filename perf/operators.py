"""What the training operators are measured on: a dense layer with its bias,
activation and residual, group norm with an activation over channels-last
arrays, and the AdamW step of a whole parameter tree.

A case names one call (forward, or forward and gradients) and its sizes;
`listed` are the fixed ones, `draw` more of the same ranges.  `run` computes a
case in plain torch operations, or, with `own`, through jax4j_b200's entry
points; `exact` computes it in 64 bits from the definitions.
"""
import math

import torch

own = False

ACTIVATIONS = ("none", "relu", "tanh", "sigmoid", "silu", "gelu")
GELU_C = math.sqrt(2.0 / math.pi)
GELU_A = 0.044715
EPS_NORM = 1e-5
LR, BETA1, BETA2, EPS, DECAY = 1e-3, 0.9, 0.999, 1e-8, 0.01
BLOCK = 128          # elements that share one step of an 8-bit moment
TOP_M, TOP_R = 448.0, 480.0  # largest code value of a first moment, of a second moment's root
TINY = 2.0 ** -100   # a block whose largest moment is below it is held as zeros


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # a hidden layer for one request: bound by reading the weight and by the call itself
        dict(name="dense one row", op="dense", M=1, K=4096, N=4096, act="silu", bias=True, residual=False,
             train=False, f64=False),
        # the hidden layer of the 784-512-10 tanh network, forward and gradients
        dict(name="dense tanh 256 train", op="dense", M=256, K=784, N=512, act="tanh", bias=True, residual=False,
             train=True, f64=False),
        # a hidden layer of the 4-layer network at its batch of 8192, as a residual block
        dict(name="dense gelu 8192 residual", op="dense", M=8192, K=4096, N=4096, act="gelu", bias=True,
             residual=True, train=False, f64=False),
        # forward and gradients where no size fills a tile
        dict(name="dense odd train", op="dense", M=4099, K=1000, N=2050, act="gelu", bias=True, residual=True,
             train=True, f64=False),
        # a small array in double precision
        dict(name="norm small f64", op="norm", B=4, S=300, C=96, G=6, act="silu", affine=True, train=False, f64=True),
        # feature maps of 64 x 64 with 10 channels to a group, forward
        dict(name="norm maps", op="norm", B=8, S=4096, C=320, G=32, act="silu", affine=True, train=False, f64=False),
        # odd feature maps, forward and gradients
        dict(name="norm maps odd train", op="norm", B=5, S=3021, C=250, G=10, act="silu", affine=True, train=True,
             f64=False),
        # hidden rows of the 4-layer network, one group a row (layer norm), forward and gradients
        dict(name="norm rows train", op="norm", B=8192, S=1, C=4096, G=1, act="none", affine=True, train=True,
             f64=False),
        # the 784-512-10 network: four leaves, bound by the call
        dict(name="adamw 784-512-10", op="adamw", sizes="401408,512,5120,10", bits=32, f64=False, step=7),
        # the 1024-4096-4096-4096-1000 network, moments in the weights' type
        dict(name="adamw mlp4", op="adamw", sizes="4194304,4096,16777216,4096,16777216,4096,4096000,1000", bits=32,
             f64=False, step=1000),
        # the same network, moments in 8 bits
        dict(name="adamw mlp4 8 bit", op="adamw", sizes="4194304,4096,16777216,4096,16777216,4096,4096000,1000",
             bits=8, f64=False, step=1000),
        # leaves of every odd size, moments in 8 bits
        dict(name="adamw ragged 8 bit", op="adamw",
             sizes="1,3,127,129,1000,4097,65537,250001,77,1048573,333,12345,640000,31,524289,999", bits=8, f64=False,
             step=1),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("dense", "norm", "adamw"))
    f64 = rng.random() < 0.15
    train = rng.random() < 0.55
    # relu's slope jumps at 0: a pre-activation within rounding of it has either slope, so gradients of two
    # correct evaluations differ by whole elements and say nothing
    act = rng.choice([a for a in ACTIVATIONS if not (train and a == "relu")])
    if op == "dense":
        while True:
            M, K, N = _log_int(rng, 1, 8192), _log_int(rng, 1, 4096), _log_int(rng, 1, 4096)
            if M * K * N * (3 if train else 1) <= (1 << (32 if f64 else 36)):
                break
        return dict(op=op, M=M, K=K, N=N, act=act, bias=rng.random() < 0.8, residual=rng.random() < 0.5, train=train,
                    f64=f64)
    if op == "norm":
        G = rng.choice((1, 2, 3, 5, 8, 16, 25, 32))
        while True:
            B, S, C = _log_int(rng, 1, 8192), _log_int(rng, 1, 16384), G * _log_int(rng, 1, max(1, 4096 // G))
            # below some 16 values to a group its gradient is the difference of nearly equal numbers
            if B * S * C <= (1 << (23 if f64 else 25)) and S * C >= 16 * G:
                break
        return dict(op=op, B=B, S=S, C=C, G=G, act=act, affine=rng.random() < 0.85, train=train, f64=f64)
    while True:
        sizes = [_log_int(rng, 1, 4000000) for _ in range(rng.randint(1, 20))]
        if sum(sizes) <= 40000000:
            break
    return dict(op=op, sizes=",".join(map(str, sizes)), bits=32 if f64 else rng.choice((8, 32)), f64=f64,
                step=_log_int(rng, 1, 100000))


def _dtype(case):
    return torch.float64 if case["f64"] else torch.float32


def _sizes(case):
    return [int(n) for n in case["sizes"].split(",")]


def work(case):
    e = 8 if case["f64"] else 4
    if case["op"] == "dense":
        M, K, N = case["M"], case["K"], case["N"]
        vec, res = N * case["bias"], M * N * case["residual"]
        if not case["train"]:
            return {"bytes": e * (M * K + K * N + vec + res + M * N), "flops": 2 * M * N * K}
        # x, w, bias, residual, dy read; y and the gradients of x, w and bias written (the residual's is dy)
        return {"bytes": e * (2 * M * K + 2 * K * N + 2 * vec + res + 2 * M * N), "flops": 6 * M * N * K}
    if case["op"] == "norm":
        n, c = case["B"] * case["S"] * case["C"], 2 * case["C"] * case["affine"]
        return {"bytes": e * ((4 * n + 2 * c) if case["train"] else (2 * n + c)), "flops": (40 if case["train"] else 12) * n}
    n = sum(_sizes(case))
    if case["bits"] == 32:
        return {"bytes": 7 * e * n, "flops": 18 * n}
    # weights, gradients and packed moments read; weights, packed moments and their values written
    return {"bytes": 20 * n + 2 * 4 * sum(_packed_words(k) for k in _sizes(case)), "flops": 60 * n}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    dt = _dtype(case)

    def normal(*shape, scale=1.0, shift=0.0):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=dt) * scale + shift

    s = {"case": dict(case)}
    if case["op"] == "dense":
        M, K, N = case["M"], case["K"], case["N"]
        s["x"] = normal(M, K)
        s["w"] = (torch.rand(K, N, generator=gen, device="cuda", dtype=dt) * 2 - 1) * math.sqrt(6.0 / (K + N))
        s["bias"] = normal(N, scale=0.1) if case["bias"] else None
        s["residual"] = normal(M, N) if case["residual"] else None
        s["dy"] = normal(M, N, scale=1.0 / math.sqrt(M)) if case["train"] else None
    elif case["op"] == "norm":
        B, S, C = case["B"], case["S"], case["C"]
        # activations with a mean and a spread of each channel's own
        s["x"] = normal(B, S, C) * (0.5 + torch.rand(C, generator=gen, device="cuda", dtype=dt)) + normal(C)
        s["gamma"] = normal(C, scale=0.2, shift=1.0) if case["affine"] else None
        s["beta"] = normal(C, scale=0.2) if case["affine"] else None
        s["dy"] = normal(B, S, C) if case["train"] else None
    else:
        sizes, t = _sizes(case), case["step"] - 1
        s["w"] = [normal(n, scale=0.05) for n in sizes]
        s["g"] = [normal(n, scale=1e-3) * torch.exp(normal(n)) for n in sizes]
        warm = 0.0 if t == 0 else 1.0
        m = [normal(n, scale=3e-4 * warm) for n in sizes]
        v = [(normal(n, scale=1e-3 * warm) * torch.exp(0.5 * normal(n))).square() for n in sizes]
        # steps taken, and the betas to that power
        s["step"] = torch.tensor([float(t), BETA1 ** t, BETA2 ** t], dtype=torch.float64, device="cuda")
        s["moments"] = ([x for pair in zip(m, v) for x in pair] if case["bits"] == 32 else
                        [_pack(a, b.sqrt()) for a, b in zip(m, v)])
    return s


# ---------------------------------------------------------------------------
# 8-bit moments.  A leaf of n elements is cut into blocks of 128.  A block's
# first moments are 4-bit-exponent, 3-bit-fraction floats (sign included),
# the roots of its second moments unsigned floats of 4 and 4 bits, each times
# the block's step = largest value / largest code.  A leaf is one array of
# 32-bit words: the codes of the first moments, those of the roots, the steps
# of the first moments, the steps of the roots.
# ---------------------------------------------------------------------------
def _packed_words(n):
    return (2 * (BLOCK // 4) + 2) * ((n + BLOCK - 1) // BLOCK)


def _blocks(x):
    return torch.nn.functional.pad(x, (0, -x.numel() % BLOCK)).view(-1, BLOCK)


def _scaled(x, top_code):
    top = x.abs().amax(1, keepdim=True)
    held = top >= TINY
    inv = torch.where(held, top_code / top, torch.zeros_like(top))
    return x * inv, torch.where(held, top / top_code, torch.zeros_like(top))


def _pack(m, r):
    ym, step_m = _scaled(_blocks(m), TOP_M)
    code_m = ym.to(torch.float8_e4m3fn).view(torch.uint8)
    yr, step_r = _scaled(_blocks(r), TOP_R)
    bits = yr.view(torch.int32)
    normal = (((bits + 0x3FFFF + ((bits >> 19) & 1)) >> 19) - (120 << 4)).clamp(max=254)
    small = torch.maximum(torch.round(yr * 1024.0).to(torch.int32), (yr > 0).to(torch.int32))  # never rounded to 0
    code_r = torch.where(yr < 2.0 ** -6, small, normal).to(torch.uint8)
    return torch.cat([code_m.reshape(-1).view(torch.int32), code_r.reshape(-1).view(torch.int32),
                      step_m.reshape(-1).view(torch.int32), step_r.reshape(-1).view(torch.int32)])


def _unpack(q, n):
    nb = (n + BLOCK - 1) // BLOCK
    words = nb * (BLOCK // 4)
    code_m, code_r = q[:words].view(torch.uint8), q[words:2 * words].view(torch.uint8)
    step_m, step_r = q[2 * words:2 * words + nb].view(torch.float32), q[2 * words + nb:].view(torch.float32)
    m = code_m.view(torch.float8_e4m3fn).to(torch.float32).view(nb, BLOCK) * step_m[:, None]
    r = (code_r.to(torch.int32) << 19).view(torch.float32) * 2.0 ** 120
    r = r.view(nb, BLOCK) * step_r[:, None]
    return m.reshape(-1)[:n], r.reshape(-1)[:n]


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _act(u, name):
    if name == "relu":
        return torch.where(u > 0, u, torch.zeros_like(u))
    if name == "tanh":
        return torch.tanh(u)
    if name == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-u))
    if name == "silu":
        return u / (1.0 + torch.exp(-u))
    if name == "gelu":  # the tanh form
        return 0.5 * u * (1.0 + torch.tanh(GELU_C * (u + GELU_A * u * u * u)))
    return u


def _act_slope(u, name):
    if name == "relu":
        return (u > 0).to(u.dtype)
    if name == "tanh":
        t = torch.tanh(u)
        return 1.0 - t * t
    if name == "sigmoid":
        s = 1.0 / (1.0 + torch.exp(-u))
        return s * (1.0 - s)
    if name == "silu":
        s = 1.0 / (1.0 + torch.exp(-u))
        return s * (1.0 + u * (1.0 - s))
    if name == "gelu":
        t = torch.tanh(GELU_C * (u + GELU_A * u * u * u))
        return 0.5 * (1.0 + t) + 0.5 * u * (1.0 - t * t) * GELU_C * (1.0 + 3.0 * GELU_A * u * u)
    return torch.ones_like(u)


def _plain_dense(s, case):
    z = s["x"] @ s["w"]
    if s["bias"] is not None:
        z = z + s["bias"]
    y = _act(z, case["act"])
    if s["residual"] is not None:
        y = y + s["residual"]
    if not case["train"]:
        return {"y": y}
    dz = s["dy"] * _act_slope(z, case["act"])
    out = {"y": y, "dx": dz @ s["w"].T, "dw": s["x"].T @ dz}
    if s["bias"] is not None:
        out["dbias"] = dz.sum(0)
    if s["residual"] is not None:
        out["dresidual"] = s["dy"]
    return out


def _plain_norm(s, case):
    B, S, C, G = case["B"], case["S"], case["C"], case["G"]
    x = s["x"].view(B, S, G, C // G)
    mean = x.mean((1, 3), keepdim=True)
    d = x - mean
    rstd = 1.0 / torch.sqrt((d * d).mean((1, 3), keepdim=True) + EPS_NORM)
    xhat = (d * rstd).view(B, S, C)
    u = xhat * s["gamma"] + s["beta"] if case["affine"] else xhat
    y = _act(u, case["act"])
    if not case["train"]:
        return {"y": y}
    du = s["dy"] * _act_slope(u, case["act"])
    out = {"y": y}
    if case["affine"]:
        out["dgamma"], out["dbeta"] = (du * xhat).sum((0, 1)), du.sum((0, 1))
        du = du * s["gamma"]
    h, xg = du.view(B, S, G, C // G), xhat.view(B, S, G, C // G)
    dx = rstd * (h - h.mean((1, 3), keepdim=True) - xg * (h * xg).mean((1, 3), keepdim=True))
    out["dx"] = dx.view(B, S, C)
    return out


def _plain_adamw_leaf(w, g, m, v, p1, p2):
    """One leaf's new weights and moments; the products are rounded one by one."""
    m = m.mul(BETA1).add(g.mul(1.0 - BETA1))
    v = v.mul(BETA2).add(g.mul(g).mul(1.0 - BETA2))
    r = v.sqrt()
    scale_m, scale_r = (1.0 / (1.0 - p1)).to(w.dtype), (1.0 / torch.sqrt(1.0 - p2)).to(w.dtype)
    update = m.mul(scale_m).div(r.mul(scale_r).add(EPS))
    return w.sub(w.mul(LR * DECAY)).sub(update.mul(LR)), m, v, r


def _plain_adamw(s, case):
    step = torch.stack([s["step"][0] + 1.0, s["step"][1] * BETA1, s["step"][2] * BETA2])
    q = s["moments"]
    if case["bits"] == 32:
        new = [_plain_adamw_leaf(w, g, q[2 * i], q[2 * i + 1], step[1], step[2])
               for i, (w, g) in enumerate(zip(s["w"], s["g"]))]
        return {"step": step, "w": [n[0] for n in new], "m": [n[1] for n in new], "v": [n[2] for n in new]}
    old = [_unpack(p, w.numel()) for p, w in zip(q, s["w"])]
    new = [_plain_adamw_leaf(w, g, m, r * r, step[1], step[2]) for w, g, (m, r) in zip(s["w"], s["g"], old)]
    held = [_unpack(_pack(n[1], n[3]), n[0].numel()) for n in new]
    return {"step": step, "w": [n[0] for n in new], "m": [h[0] for h in held], "v": [h[1] * h[1] for h in held]}


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------
def _array(J, t):
    return J.ConcreteNDArray(t, tuple(t.shape))


def _tensor(a):
    return a.tensor().view(a.shape().dimensions())


def _own_dense(J, s, case):
    names = [n for n in ("x", "w", "bias", "residual") if s[n] is not None]
    args = [_array(J, s[n]) for n in names]

    def layer(*a):
        d = dict(zip(names, a))
        return J.Nn.dense(d["x"], d["w"], bias=d.get("bias"), activation=case["act"], residual=d.get("residual"))

    if not case["train"]:
        return {"y": _tensor(layer(*args))}
    y, pull = J.JAX.vjp(layer, *args)
    grads = pull(_array(J, s["dy"]))
    return {"y": _tensor(y), **{"d" + n: _tensor(g) for n, g in zip(names, grads)}}


def _own_norm(J, s, case):
    names = [n for n in ("x", "gamma", "beta") if s[n] is not None]
    args = [_array(J, s[n]) for n in names]

    def norm(*a):
        d = dict(zip(names, a))
        return J.Nn.groupNorm(d["x"], case["G"], d.get("gamma"), d.get("beta"), eps=EPS_NORM, activation=case["act"])

    if not case["train"]:
        return {"y": _tensor(norm(*args))}
    y, pull = J.JAX.vjp(norm, *args)
    grads = pull(_array(J, s["dy"]))
    return {"y": _tensor(y), **{"d" + n: _tensor(g) for n, g in zip(names, grads)}}


def _own_adamw(J, s, case):
    params = J.PyTree.list(*[J.PyTree.leaf(_array(J, w)) for w in s["w"]])
    grads = J.PyTree.list(*[J.PyTree.leaf(_array(J, g)) for g in s["g"]])
    state = J.AdamWState(params, case["bits"], _array(J, s["step"]), [_array(J, q) for q in s["moments"]])
    params, state = J.Optim.adamW(params, grads, state, LR, beta1=BETA1, beta2=BETA2, eps=EPS, weightDecay=DECAY)
    m, v = state.moments()
    flat = [[_tensor(a) for a in J.PyTrees.flatten(t)] for t in (params, m, v)]
    return {"step": _tensor(state.step()), "w": flat[0], "m": flat[1], "v": flat[2]}


def run(state):
    case = state["case"]
    if own:
        import jax4j_b200 as J
        return {"dense": _own_dense, "norm": _own_norm, "adamw": _own_adamw}[case["op"]](J, state, case)
    return {"dense": _plain_dense, "norm": _plain_norm, "adamw": _plain_adamw}[case["op"]](state, case)


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _exact_act(u, name):
    """act(u) and its derivative."""
    if name == "none":
        return u, torch.ones_like(u)
    if name == "relu":
        return u.clamp(min=0), torch.heaviside(u, torch.zeros((), dtype=u.dtype, device=u.device))
    if name == "tanh":
        return torch.tanh(u), torch.cosh(u.clamp(-300, 300)) ** -2
    if name == "sigmoid":
        return torch.sigmoid(u), torch.sigmoid(u) * torch.sigmoid(-u)
    # u sigmoid(k(u)): k = u (silu), or 2 GELU_C (u + GELU_A u^3) (gelu: 1 + tanh(a) = 2 sigmoid(2a))
    k = u if name == "silu" else 2 * GELU_C * (u + GELU_A * u ** 3)
    dk = torch.ones_like(u) if name == "silu" else 2 * GELU_C * (1 + 3 * GELU_A * u ** 2)
    return u * torch.sigmoid(k), torch.sigmoid(k) + u * torch.sigmoid(k) * torch.sigmoid(-k) * dk


def _exact_dense(s, case):
    x, w = s["x"].double(), s["w"].double()
    z = torch.einsum("mk,kn->mn", x, w) + (0 if s["bias"] is None else s["bias"].double()[None, :])
    y, slope = _exact_act(z, case["act"])
    out = {"y": y if s["residual"] is None else s["residual"].double() + y}
    if case["train"]:
        dz = slope * s["dy"].double()
        out["dx"] = torch.einsum("mn,kn->mk", dz, w)
        out["dw"] = torch.einsum("mk,mn->kn", x, dz)
        if s["bias"] is not None:
            out["dbias"] = torch.einsum("mn->n", dz)
        if s["residual"] is not None:
            out["dresidual"] = s["dy"].double()
    return out


def _exact_norm(s, case):
    B, S, C, G = case["B"], case["S"], case["C"], case["G"]
    # [B, G, elements of the group]
    groups = lambda t: t.double().reshape(B, S, G, C // G).transpose(1, 2).reshape(B, G, -1)  # noqa: E731
    back = lambda t: t.reshape(B, G, S, C // G).transpose(1, 2).reshape(B, S, C)  # noqa: E731
    x = groups(s["x"])
    var, mean = torch.var_mean(x, 2, correction=0, keepdim=True)
    sd = torch.sqrt(var + EPS_NORM)
    xhat = back((x - mean) / sd)
    gamma = s["gamma"].double() if case["affine"] else torch.ones(C, dtype=torch.float64, device="cuda")
    beta = s["beta"].double() if case["affine"] else torch.zeros(C, dtype=torch.float64, device="cuda")
    y, slope = _exact_act(torch.addcmul(beta, xhat, gamma), case["act"])
    out = {"y": y}
    if case["train"]:
        du = slope * s["dy"].double()
        if case["affine"]:
            out["dgamma"], out["dbeta"] = torch.einsum("bsc,bsc->c", du, xhat), torch.einsum("bsc->c", du)
        h, xg = groups(du * gamma), groups(xhat)
        # the part of h along neither 1 nor xhat, over the standard deviation
        dx = (h - h.mean(2, keepdim=True) - xg * torch.einsum("bgk,bgk->bg", h, xg)[..., None] / h.shape[2]) / sd
        out["dx"] = back(dx)
    return out


def _exact_adamw(s, case):
    t, q = case["step"], s["moments"]
    out = {"step": torch.tensor([t, BETA1 ** t, BETA2 ** t], dtype=torch.float64), "w": [], "m": [], "v": []}
    for i, (w, g) in enumerate(zip(s["w"], s["g"])):
        n, g = w.numel(), g.double()
        if case["bits"] == 32:
            m, v = q[2 * i].double(), q[2 * i + 1].double()
        else:
            nb = -(-n // BLOCK)
            codes = q[i][:nb * BLOCK // 2].view(torch.uint8).long().view(2, nb, BLOCK)
            steps = q[i][nb * BLOCK // 2:].view(torch.float32).double().view(2, nb, 1)
            sign, e, f = 1 - 2 * (codes[0] >> 7), (codes[0] >> 3) & 15, codes[0] & 7
            m = sign * torch.where(e > 0, (8 + f) * 2.0 ** (e - 10).double(), f * 2.0 ** -9) * steps[0]
            e, f = codes[1] >> 4, codes[1] & 15
            v = (torch.where(e > 0, (16 + f) * 2.0 ** (e - 11).double(), f * 2.0 ** -10) * steps[1]) ** 2
            m, v = m.reshape(-1)[:n], v.reshape(-1)[:n]
        m, v = torch.lerp(g, m, BETA1), torch.lerp(g ** 2, v, BETA2)
        mhat, vhat = m / (1 - BETA1 ** t), v / (1 - BETA2 ** t)
        w = w.double()
        out["w"].append(w - LR * (mhat / (vhat ** 0.5 + EPS) + DECAY * w))
        # a moment held in 8 bits is the rounding of one computed in 32: it has no value in 64
        out["m"].append(m if case["bits"] == 32 else None)
        out["v"].append(v if case["bits"] == 32 else None)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"dense": _exact_dense, "norm": _exact_norm, "adamw": _exact_adamw}[case["op"]](s, case)
