"""What is measured of the normalised layer and of the orthogonalised update of its weights.

Four operators, each in its plain form (elementary torch operations in 32 bits) and, where `own` is true,
as a user of the C ABI calls it:

  group_norm            y = act((x - mean) * rstd * weight + bias) over [batch, positions, channels], channels
                        last, mean and rstd per (sample, group); returns y and the statistics that the
                        gradient needs
  group_norm_backward   the gradients of x, weight and bias from the upstream gradient
  newton_schulz         the update matrix with its singular values driven towards one: X = G / (|G| + eps),
                        then `steps` times X = a X + (b A + c A^2) X with A = X X^T
  muon_step             a training step of several weight matrices: momentum, its Newton-Schulz
                        orthogonalisation, weight decay and the update; returns weights and momenta
"""
import ctypes
import math

import torch

own = False

DEVICE = "cuda:0"
EPS_NORM = 1e-5
EPS_NS = 1e-7
STEPS = 5
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
LEARNING_RATE, MOMENTUM, WEIGHT_DECAY = 0.02, 0.95, 0.01
ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2}


# ------------------------------------------------------------------------------------ cases

def listed():
    return [
        # the hidden layer of the 784-256-10 network, normalised, at the training batch of 256: a call of a
        # quarter of a megabyte, all latency
        {"name": "norm_mlp_256", "op": "group_norm", "batch": 256, "positions": 1, "channels": 256, "groups": 8, "act": "relu"},
        # a feature map of 64 x 64 positions, the usual 32 groups
        {"name": "norm_map", "op": "group_norm", "batch": 16, "positions": 4096, "channels": 256, "groups": 32, "act": "silu"},
        # sequences of odd length, 30 channels a group: no vector of four lies inside a group
        {"name": "norm_odd", "op": "group_norm", "batch": 5, "positions": 7031, "channels": 330, "groups": 11, "act": "none"},
        # the same network's layer at the large batch of 8192, backward: weight and bias gradients sum 8192 rows
        {"name": "norm_grad_mlp_8192", "op": "group_norm_backward", "batch": 8192, "positions": 1, "channels": 256, "groups": 8, "act": "relu"},
        # a large feature map, backward
        {"name": "norm_grad_map", "op": "group_norm_backward", "batch": 32, "positions": 4096, "channels": 512, "groups": 32, "act": "silu"},
        {"name": "norm_grad_odd", "op": "group_norm_backward", "batch": 5, "positions": 7031, "channels": 330, "groups": 11, "act": "none"},
        # the output layer's gradient of the 784-256-10 network: the smallest matrix that a step updates
        {"name": "ns_head", "op": "newton_schulz", "batch": 1, "rows": 256, "cols": 10},
        # an odd tall matrix
        {"name": "ns_odd", "op": "newton_schulz", "batch": 1, "rows": 1000, "cols": 333},
        # the square sizes of the matrix product's own benchmark
        {"name": "ns_2048", "op": "newton_schulz", "batch": 1, "rows": 2048, "cols": 2048},
        {"name": "ns_4096", "op": "newton_schulz", "batch": 1, "rows": 4096, "cols": 4096},
        # the two weight matrices of the 784-256-10 network in one step
        {"name": "muon_mlp", "op": "muon_step", "shapes": "784x256,256x10", "nesterov": True},
        # a wider network's layers in one step, one of them of an odd width
        {"name": "muon_wide", "op": "muon_step", "shapes": "784x2048,2048x2048,2048x4096,4096x1001", "nesterov": True},
    ]


def _log_uniform(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["group_norm", "group_norm_backward", "newton_schulz", "muon_step"])
    if op.startswith("group_norm"):
        groups = rng.choice([1, 2, 3, 4, 8, 11, 16, 32])
        width = _log_uniform(rng, 1, 128)
        if rng.random() < 0.5:
            width = -(-width // 4) * 4                  # vectors of four lie inside a group, as in most networks
        channels = groups * width
        positions = rng.choice([1, _log_uniform(rng, 1, 16384)])
        if positions * width < 16:                      # the gradient of a group of two or three values is all cancellation
            positions = -(-16 // width)
        batch = _log_uniform(rng, 1, max(1, min(16384 if positions == 1 else 64, (1 << 26) // (positions * channels))))
        return {"op": op, "batch": batch, "positions": positions, "channels": channels, "groups": groups,
                "act": rng.choice(sorted(ACTIVATIONS))}
    if op == "newton_schulz":
        rows, cols = _log_uniform(rng, 1, 2900), _log_uniform(rng, 1, 2900)
        return {"op": op, "batch": rng.choice([1, 1, 2, 5]) if rows * cols < 1 << 20 else 1, "rows": rows, "cols": cols}
    shapes = ["%dx%d" % (_log_uniform(rng, 8, 2000), _log_uniform(rng, 8, 2000)) for _ in range(rng.randint(1, 4))]
    return {"op": op, "shapes": ",".join(shapes), "nesterov": rng.random() < 0.5}


def _shapes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split(",")]


# ------------------------------------------------------------------------------------ inputs

def _gradient(gen, rows, cols, batch=None):
    """What a backward pass leaves: a few strong directions over a floor of noise, entries of about 1e-3."""
    lead = () if batch is None else (batch,)
    rank = max(1, min(rows, cols) // 8)
    u = torch.randn(*lead, rows, rank, device=DEVICE, generator=gen) / math.sqrt(rank)
    v = torch.randn(*lead, rank, cols, device=DEVICE, generator=gen)
    return (torch.matmul(u, v) + 0.3 * torch.randn(*lead, rows, cols, device=DEVICE, generator=gen)) * 1e-3


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    s = {"op": case["op"]}
    if case["op"].startswith("group_norm"):
        n, p, c, g = case["batch"], case["positions"], case["channels"], case["groups"]
        offset = 0.5 * torch.randn(c, device=DEVICE, generator=gen)
        s["x"] = torch.randn(n, p, c, device=DEVICE, generator=gen).add_(offset)
        s["weight"] = 1.0 + 0.2 * torch.randn(c, device=DEVICE, generator=gen)
        s["bias"] = 0.2 * torch.randn(c, device=DEVICE, generator=gen)
        s["groups"], s["act"] = g, case["act"]
        if case["op"] == "group_norm_backward":
            s["dy"] = torch.randn(n, p, c, device=DEVICE, generator=gen)
            # (mean, rstd) of every sample's groups, as the forward pass left them
            stats = torch.empty(n, g, 2, device=DEVICE)
            for i in range(n) if p * c > 1 << 16 else (slice(None),):
                x = s["x"][i].double().reshape(-1, p, g, c // g)
                mean = x.mean((1, 3))
                stats[i] = torch.stack((mean, ((x - mean[:, None, :, None]).square().mean((1, 3)) + EPS_NORM).rsqrt()), -1).float()
            s["stats"] = stats
        return s
    if case["op"] == "newton_schulz":
        s["g"] = _gradient(gen, case["rows"], case["cols"], case["batch"])
        return s
    s["nesterov"] = case["nesterov"]
    s["params"], s["grads"], s["momenta"] = [], [], []
    for rows, cols in _shapes(case):
        s["params"].append(torch.randn(rows, cols, device=DEVICE, generator=gen) / math.sqrt(rows))
        s["grads"].append(_gradient(gen, rows, cols))
        s["momenta"].append(10 * _gradient(gen, rows, cols))
    return s


# ------------------------------------------------------------------------------------ the plain forms

def _plain_group_norm(s):
    x = s["x"]
    n, p, c = x.shape
    xg = x.reshape(n, p, s["groups"], c // s["groups"])
    mean = xg.mean((1, 3), keepdim=True)
    d = xg - mean
    rstd = (d.square().mean((1, 3), keepdim=True) + EPS_NORM).rsqrt()
    z = (d * rstd).reshape(n, p, c) * s["weight"] + s["bias"]
    y = z if s["act"] == "none" else z.clamp(min=0) if s["act"] == "relu" else z / (1 + torch.exp(-z))
    return y, torch.stack((mean.reshape(n, -1), rstd.reshape(n, -1)), -1)


def _plain_group_norm_backward(s):
    x, dy, w = s["x"], s["dy"], s["weight"]
    n, p, c = x.shape
    g = s["groups"]
    mean, rstd = (s["stats"][:, None, :, None, k] for k in (0, 1))
    xhat = ((x.reshape(n, p, g, c // g) - mean) * rstd).reshape(n, p, c)
    dz = dy
    if s["act"] != "none":
        z = xhat * w + s["bias"]
        if s["act"] == "relu":
            dz = dy * (z > 0)
        else:
            sig = 1 / (1 + torch.exp(-z))
            dz = dy * (sig * (1 + z * (1 - sig)))
    dbias = dz.sum((0, 1))
    dweight = (dz * xhat).sum((0, 1))
    dxhat = (dz * w).reshape(n, p, g, c // g)
    xhat = xhat.reshape(n, p, g, c // g)
    s1 = dxhat.mean((1, 3), keepdim=True)
    s2 = (dxhat * xhat).mean((1, 3), keepdim=True)
    return ((dxhat - s1 - xhat * s2) * rstd).reshape(n, p, c), dweight, dbias


def _plain_newton_schulz(g):
    a, b, c = COEFFICIENTS
    tall = g.shape[-2] > g.shape[-1]
    x = g.transpose(-1, -2).contiguous() if tall else g
    x = x / (x.double().square().sum((-1, -2), keepdim=True).sqrt() + EPS_NS).float()
    for _ in range(STEPS):
        gram = torch.matmul(x, x.transpose(-1, -2))
        x = a * x + torch.matmul(b * gram + c * torch.matmul(gram, gram), x)
    return x.transpose(-1, -2).contiguous() if tall else x


def _scale(rows, cols):
    return 0.2 * math.sqrt(max(rows, cols))


def _plain_muon(s):
    params, momenta = [], []
    for p, g, m in zip(s["params"], s["grads"], s["momenta"]):
        m = MOMENTUM * m + g
        u = g + MOMENTUM * m if s["nesterov"] else m
        o = _plain_newton_schulz(u)
        params.append(p * (1 - LEARNING_RATE * WEIGHT_DECAY) - (LEARNING_RATE * _scale(*p.shape)) * o)
        momenta.append(m)
    return params, momenta


# ------------------------------------------------------------------------------------ the framework's calls

_library = None


def _lib():
    global _library
    if _library is None:
        from ctorch_amd import capi
        library = capi.load()
        capi.check(library.ctamd_init(0))
        _library = (library, capi)
    return _library


def _stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _own_group_norm(s):
    lib, capi = _lib()
    x = s["x"]
    n, p, c = x.shape
    y = torch.empty_like(x)
    stats = torch.empty(n, s["groups"], 2, device=x.device)
    capi.check(lib.ctamd_group_norm_f32(x.data_ptr(), s["weight"].data_ptr(), s["bias"].data_ptr(), EPS_NORM, ACTIVATIONS[s["act"]],
                                        y.data_ptr(), stats.data_ptr(), n, p, c, s["groups"], _stream()))
    return y, stats


def _own_group_norm_backward(s):
    lib, capi = _lib()
    x = s["x"]
    n, p, c = x.shape
    dx, dw, db = torch.empty_like(x), torch.empty(c, device=x.device), torch.empty(c, device=x.device)
    capi.check(lib.ctamd_group_norm_backward_f32(x.data_ptr(), s["weight"].data_ptr(), s["bias"].data_ptr(), s["stats"].data_ptr(),
                                                 ACTIVATIONS[s["act"]], s["dy"].data_ptr(), dx.data_ptr(), dw.data_ptr(), db.data_ptr(),
                                                 n, p, c, s["groups"], _stream()))
    return dx, dw, db


def _own_newton_schulz(s):
    lib, capi = _lib()
    g = s["g"]
    batch, rows, cols = g.shape
    size = ctypes.c_size_t()
    capi.check(lib.ctamd_newton_schulz_workspace(rows, cols, batch, ctypes.byref(size)))
    work = torch.empty(size.value, dtype=torch.uint8, device=g.device)
    out = torch.empty_like(g)
    capi.check(lib.ctamd_newton_schulz_f32(g.data_ptr(), out.data_ptr(), rows, cols, batch, STEPS, None, EPS_NS,
                                           work.data_ptr(), size.value, _stream()))
    return out


def _own_muon(s):
    lib, capi = _lib()
    params = [torch.empty_like(p) for p in s["params"]]
    momenta = [torch.empty_like(m) for m in s["momenta"]]
    mats = (capi.MuonMatrix * len(params))(*[
        capi.MuonMatrix(p.data_ptr(), g.data_ptr(), m.data_ptr(), q.data_ptr(), r.data_ptr(), p.shape[0], p.shape[1], _scale(*p.shape))
        for p, g, m, q, r in zip(s["params"], s["grads"], s["momenta"], params, momenta)])
    options = capi.MuonOptions(LEARNING_RATE, MOMENTUM, WEIGHT_DECAY, EPS_NS, int(s["nesterov"]), STEPS, COEFFICIENTS)
    size = ctypes.c_size_t()
    capi.check(lib.ctamd_muon_workspace(mats, len(params), ctypes.byref(size)))
    work = torch.empty(size.value, dtype=torch.uint8, device=DEVICE)
    capi.check(lib.ctamd_muon_step_f32(mats, len(params), ctypes.byref(options), work.data_ptr(), size.value, _stream()))
    return params, momenta


def run(state):
    op = state["op"]
    if own:
        return {"group_norm": _own_group_norm, "group_norm_backward": _own_group_norm_backward,
                "newton_schulz": _own_newton_schulz, "muon_step": _own_muon}[op](state)
    if op == "newton_schulz":
        return _plain_newton_schulz(state["g"])
    return {"group_norm": _plain_group_norm, "group_norm_backward": _plain_group_norm_backward, "muon_step": _plain_muon}[op](state)


# ------------------------------------------------------------------------------------ work and exact results

def _ns_flops(rows, cols):
    """Per step the Gram matrix and its square are symmetric (one half is enough), the third product is not."""
    m, n = min(rows, cols), max(rows, cols)
    return STEPS * (m * (m + 1) * n + m * (m + 1) * m + 2 * m * m * n)


def work(case):
    if case["op"].startswith("group_norm"):
        n = case["batch"] * case["positions"] * case["channels"]
        small = 4 * case["channels"] + 8 * case["batch"] * case["groups"]
        if case["op"] == "group_norm":
            return {"bytes": 8 * n + 2 * small, "flops": 8 * n}
        return {"bytes": 12 * n + 4 * small, "flops": 16 * n}
    if case["op"] == "newton_schulz":
        n = case["batch"] * case["rows"] * case["cols"]
        return {"bytes": 8 * n, "flops": case["batch"] * _ns_flops(case["rows"], case["cols"]) + 4 * n}
    shapes = _shapes(case)
    n = sum(r * c for r, c in shapes)
    return {"bytes": 20 * n, "flops": sum(_ns_flops(r, c) for r, c in shapes) + 12 * n}


def _exact_newton_schulz(g):
    """On the eigenvalues' side: with A = X X^T, W = a + b A + c A^2 and W, A commuting, the next Gram matrix is
    W A W; the product Q of the W's is applied to the first X once."""
    a, b, c = COEFFICIENTS
    x = g.double()
    x = x / (torch.linalg.matrix_norm(x, keepdim=True) + EPS_NS)
    if g.shape[-2] > g.shape[-1]:
        x = x.mT.contiguous()
    gram = x @ x.mT.contiguous()
    q = eye = torch.eye(x.shape[-2], dtype=torch.float64, device=x.device)
    for k in range(STEPS):
        w = a * eye + gram @ (b * eye + c * gram)
        q = w @ q
        gram = w @ (gram @ w)
    x = q @ x
    return x.mT.contiguous() if g.shape[-2] > g.shape[-1] else x


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "newton_schulz":
        return _exact_newton_schulz(s["g"])
    if case["op"] == "muon_step":
        params, momenta = [], []
        for p, g, m in zip(s["params"], s["grads"], s["momenta"]):
            p, g, m = p.double(), g.double(), m.double()
            buf = g + MOMENTUM * m
            o = _exact_newton_schulz(g + MOMENTUM * buf if s["nesterov"] else buf)
            params.append(p - LEARNING_RATE * (WEIGHT_DECAY * p + _scale(*p.shape) * o))
            momenta.append(buf)
        return params, momenta
    n, p, c = s["x"].shape
    x = s["x"].double().reshape(n, p, s["groups"], -1).transpose(1, 2)          # [n, groups, positions, width]
    w, b = s["weight"].double(), s["bias"].double()
    if case["op"] == "group_norm":
        var, mean = torch.var_mean(x, (2, 3), correction=0, keepdim=True)
        rstd = 1 / torch.sqrt(var + EPS_NORM)
        z = torch.addcmul(b, ((x - mean) * rstd).transpose(1, 2).reshape(n, p, c), w)
        y = {"none": lambda: z, "relu": lambda: torch.relu(z), "silu": lambda: z * torch.sigmoid(z)}[s["act"]]()
        return y, torch.stack((mean.reshape(n, -1), rstd.reshape(n, -1)), -1)
    # from the definition: y's derivative along x through the mean and the deviation, as products of sums
    mean, rstd = s["stats"].double()[:, :, None, None, :].unbind(-1)
    h = ((x - mean) * rstd).transpose(1, 2).reshape(n, p, c)
    up = s["dy"].double()
    if s["act"] == "relu":
        up = torch.where(torch.addcmul(b, h, w) > 0, up, torch.zeros_like(up))
    elif s["act"] == "silu":
        z = torch.addcmul(b, h, w)
        sig = torch.sigmoid(z)
        up = up * torch.addcmul(sig, z * sig, 1 - sig)
    along_c, along_h = up.sum(1), (up * h).sum(1)                               # [n, channels]
    width = c // s["groups"]
    per = lambda v: ((v * w).reshape(n, -1, width).sum(-1) / (p * width)).repeat_interleave(width, 1)[:, None]  # noqa: E731
    r = rstd.reshape(n, 1, -1).repeat_interleave(width, 2)
    return (up * w - per(along_c) - h * per(along_h)) * r, along_h.sum(0), along_c.sum(0)
