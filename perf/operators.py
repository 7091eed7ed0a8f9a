"""The cases of the 8-bit product and of the Muon update: what they are given, what they return, and what they cannot do without.

Four operators:
  product        rows of 8-bit integers against rows of 8-bit integers, with a scale for each row of either side
  volume         the all-pairs correlation volume of feature maps that are quantised on the way in (a scale for each pixel)
  orthogonalize  a list of matrices, each turned towards its nearest semi-orthogonal one by five quintic Newton-Schulz steps
  step           one step of the Muon optimiser: momentum, Nesterov, orthogonalisation, decay and update of every filter

`own` false: elementary torch operations.  `own` true: the framework's own entry points, as a user calls them."""
import math

import torch

own = False

STEPS, COEFFICIENTS, EPS = 5, (3.4445, -4.7750, 2.0315), 1e-7
LR, DECAY, MOMENTUM = 1e-4, 1e-4, 0.95        # learning rate and decay of the framework's training configuration

# Filters (rows = output channels, columns = input channels x window) of the event model with four event targets and degree 2, and of its
# update block alone.
MODEL = ("64x245*2,64x576*8,64x1152,96x64*2,96x576*2,96x864*6,128x96*2,128x196,128x864*2,128x1152*6,128x1920*6,"
         "256x128*2,256x567,256x1152*2,576x256,4x2304,124x2304,192x2304")
UPDATE_BLOCK = "256x567,192x2304,128x196,64x1152,124x2304,128x1920*6,256x1152*2,4x2304,576x256"


def listed():
    return [
        # The latency of one call: a user who orthogonalises a single filter of the encoder.
        {"name": "orthogonalize one filter", "op": "orthogonalize", "shapes": "64x576", "dtype": "float32"},
        # Every filter of the model, as one training step needs them.
        {"name": "orthogonalize model", "op": "orthogonalize", "shapes": MODEL, "dtype": "float32"},
        # Sizes that fit no tile, rows alone, tall and wide, in 16 bits.
        {"name": "orthogonalize ragged", "op": "orthogonalize", "shapes": "1x77,37x1000,517x131,300x300,513x129,2x2049", "dtype": "bfloat16"},
        # The largest matrix: the work is three products in a row, five times.
        {"name": "orthogonalize large", "op": "orthogonalize", "shapes": "4096x4096", "dtype": "bfloat16"},
        # A training step of the update block: parameters, gradients and momentum in 32 bits.
        {"name": "step update block", "op": "step", "shapes": UPDATE_BLOCK},
        # A training step of wide layers.
        {"name": "step wide layers", "op": "step", "shapes": "1024x1024*4,1024x4096*2"},
        # A single token against a square layer: every weight is read once, nothing is reused.
        {"name": "product one token", "op": "product", "batch": 1, "shared": True, "m": 1, "n": 4096, "k": 4096, "out": "bfloat16"},
        # One row for each pixel of a 60 x 80 map through the motion encoder's first layer (567 look-up channels: an odd row length).
        {"name": "product pixels", "op": "product", "batch": 1, "shared": True, "m": 4800, "n": 256, "k": 567, "out": "float32"},
        # Odd in every size, several matrices in a call, each with its own right side.
        {"name": "product ragged", "op": "product", "batch": 3, "shared": False, "m": 333, "n": 1001, "k": 1021, "out": "float16"},
        # Bound by the matrix instructions.
        {"name": "product large", "op": "product", "batch": 1, "shared": True, "m": 8192, "n": 8192, "k": 8192, "out": "bfloat16"},
        # The correlation volume at 640 x 480 with four event targets, stored in 16 bits: as a forward pass builds it.
        {"name": "volume 60x80", "op": "volume", "batch": 1, "targets": 4, "dim": 256, "h": 60, "w": 80, "out": "float16"},
        # A map that fits no tile of the look-up's layout, two samples, stored in 32 bits.
        {"name": "volume ragged", "op": "volume", "batch": 2, "targets": 1, "dim": 128, "h": 47, "w": 61, "out": "float32"},
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("orthogonalize", "step", "product", "volume"))
    if op in ("orthogonalize", "step"):
        count = _log(rng, 1, 30)
        most = 2048 if count <= 4 else 640
        shapes = ",".join("%dx%d" % (_log(rng, 1, most), _log(rng, 1, most)) for _ in range(count))
        case = {"op": op, "shapes": shapes}
        if op == "orthogonalize":
            case["dtype"] = rng.choice(("float32", "bfloat16", "float16"))
        return case
    if op == "product":
        batch = rng.choice((1, 1, 2, 5))
        return {"op": op, "batch": batch, "shared": rng.random() < 0.5, "m": _log(rng, 1, 8192 // batch), "n": _log(rng, 1, 8192), "k": _log(rng, 1, 8192),
                "out": rng.choice(("float32", "bfloat16", "float16"))}
    return {"op": op, "batch": rng.choice((1, 2)), "targets": rng.randint(1, 4), "dim": rng.choice((64, 128, 192, 256)), "h": rng.randint(8, 72), "w": rng.randint(8, 90),
            "out": rng.choice(("float32", "float16"))}


def _sizes(case):
    sizes = []
    for part in case["shapes"].split(","):
        shape, _, times = part.partition("*")
        m, n = shape.split("x")
        sizes += [(int(m), int(n))] * int(times or 1)
    return sizes


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(1_000_003 * (seed + 1))


def _gradient(m, n, g, size):
    """A matrix as a gradient is one: a few strong directions, a long tail of weak ones, and noise."""
    r = max(1, min(m, n) // 4)
    left = torch.randn((m, r), generator=g, device="cuda") * torch.logspace(0, -3, r, device="cuda")
    right = torch.randn((r, n), generator=g, device="cuda")
    return size * (left @ right + 0.03 * torch.randn((m, n), generator=g, device="cuda"))


def prepare(case, seed):
    g = _generator(seed)
    if case["op"] == "orthogonalize":
        kind = getattr(torch, case["dtype"])
        return {"case": case, "x": [_gradient(m, n, g, 1e-3).to(kind) for m, n in _sizes(case)]}
    if case["op"] == "step":
        sizes = _sizes(case)
        weights = [torch.nn.Parameter(torch.randn((m, n), generator=g, device="cuda") / math.sqrt(n)) for m, n in sizes]
        for p, (m, n) in zip(weights, sizes):
            p.grad = _gradient(m, n, g, 1e-3)
        return {"case": case, "weights": weights, "momentum": [_gradient(m, n, g, 1e-2) for m, n in sizes]}
    if case["op"] == "product":
        def rows(r):
            shape = (case["batch"], r) if case["batch"] > 1 else (r,)
            q = torch.randn(shape + (case["k"],), generator=g, device="cuda").mul_(40).round_().clamp_(-127, 127).to(torch.int8)
            return q, 0.01 * torch.randn(shape, generator=g, device="cuda").exp_()
        a, sa = rows(case["m"])
        b, sb = rows(case["n"])
        if case["shared"] and case["batch"] > 1:
            b, sb = b[0], sb[0]
        return {"case": case, "a": a, "sa": sa, "b": b, "sb": sb}
    shape = (case["dim"], case["h"], case["w"])

    def maps(*lead):
        loud = torch.randn(lead + (1,) + shape[1:], generator=g, device="cuda").mul_(0.5).exp_()
        return loud * torch.randn(lead + shape, generator=g, device="cuda")
    return {"case": case, "reference": maps(case["batch"]), "target": maps(case["targets"], case["batch"])}


# ---------------------------------------------------------------------------------------------------------------------------- plain forms
def _orthogonal(x):
    """x (m, n) in 32 bits -> the Newton-Schulz iterate of x / |x| after STEPS steps.  The norm is summed in 64 bits."""
    a, b, c = COEFFICIENTS
    x = x / (x.double().square().sum().sqrt() + EPS).float()
    tall = x.shape[0] > x.shape[1]
    x = x.t().contiguous() if tall else x
    for _ in range(STEPS):
        gram = x @ x.t()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.t().contiguous() if tall else x


def _stepped(p, grad, momentum):
    m, n = p.shape
    momentum.mul_(MOMENTUM).add_(grad)
    update = _orthogonal(grad + MOMENTUM * momentum)
    p.mul_(1 - LR * DECAY).sub_(update, alpha=LR * 0.2 * math.sqrt(max(m, n)))


def _quantised(f):
    """f (..., D, h, w) -> whole numbers (..., D, h * w) in -127 .. 127 and the scale of each pixel (..., 1, h * w).  The quotient is taken in
    64 bits: in 32, values next to a half would be rounded the wrong way."""
    f = f.flatten(-2)
    most = f.abs().amax(-2, keepdim=True)
    return torch.where(most > 0, torch.round(f.double() * 127 / most), 0.0).float(), most / 127


def _tiled(v, h, w):
    """(..., h * w) -> (..., tiles * 32): the plane as 4 x 8 tiles in row order, edge tiles filled up with zeros."""
    lead, th, tw = v.shape[:-1], -(-h // 4), -(-w // 8)
    v = torch.nn.functional.pad(v.reshape(*lead, h, w), (0, tw * 8 - w, 0, th * 4 - h))
    return v.reshape(*lead, th, 4, tw, 8).transpose(-3, -2).reshape(*lead, th * tw * 32)


def run(state):
    case = state["case"]
    if case["op"] == "orthogonalize":
        if own:
            from bflow_amd import muon
            return muon.orthogonalize(state["x"])
        return [_orthogonal(x.float()).to(x.dtype) for x in state["x"]]
    if case["op"] == "step":
        weights, momentum = state["weights"], state["momentum"]
        if own:
            if "optimizer" not in state:
                from bflow_amd import muon
                state["optimizer"] = muon.Muon(weights, lr=LR, weight_decay=DECAY, momentum=MOMENTUM)
                for p, v in zip(weights, momentum):
                    state["optimizer"].state[p]["momentum_buffer"] = v
            state["optimizer"].step()
        else:
            with torch.no_grad():
                for p, v in zip(weights, momentum):
                    _stepped(p, p.grad, v)
        return {"weights": weights, "momentum": momentum}
    if case["op"] == "product":
        kind = getattr(torch, case["out"])
        if own:
            from bflow_amd import int8
            return int8.matmul(state["a"], state["sa"], state["b"], state["sb"], out_dtype=kind)
        sums = state["a"].float() @ state["b"].float().transpose(-1, -2)
        return (sums * state["sa"].unsqueeze(-1) * state["sb"].unsqueeze(-2)).to(kind)
    reference, target = state["reference"], state["target"]
    kind = getattr(torch, case["out"])
    if own:
        from bflow_amd.corr import CorrComputation
        pairs = CorrComputation(reference, target, [1] * case["targets"])
        return pairs.get_correlation_volume(tiled=True, precision="i8" if kind == torch.float16 else "i8/w")
    (q1, s1), (q2, s2) = _quantised(reference), _quantised(target)
    sums = q1.transpose(-1, -2).contiguous() @ q2
    volume = sums * (s1.transpose(-1, -2) / math.sqrt(case["dim"])) * s2
    return _tiled(volume, case["h"], case["w"]).to(kind)


# ---------------------------------------------------------------------------------------------------------------------------------- work
def work(case):
    if case["op"] in ("orthogonalize", "step"):
        size = 20 if case["op"] == "step" else 2 * getattr(torch, case["dtype"]).itemsize
        total = {"bytes": 0, "flops": 0}
        for m, n in _sizes(case):
            r, s = min(m, n), max(m, n)
            total["bytes"] += size * m * n
            total["flops"] += STEPS * (r * (r + 1) * s + r * r * (r + 1) + 2 * r * r * s)   # the two symmetric products: half of each
        return total
    out = getattr(torch, case["out"]).itemsize
    if case["op"] == "product":
        b, m, n, k = (case[x] for x in ("batch", "m", "n", "k"))
        right = 1 if case["shared"] else b
        return {"bytes": b * m * (k + 4) + right * n * (k + 4) + b * m * n * out, "flops": 2 * b * m * n * k}
    pixels, plane = case["h"] * case["w"], -(-case["h"] // 4) * -(-case["w"] // 8) * 32
    b, t, d = case["batch"], case["targets"], case["dim"]
    return {"bytes": 4 * d * pixels * b * (1 + t) + t * b * pixels * plane * out, "flops": 2 * t * b * d * pixels * pixels}


# --------------------------------------------------------------------------------------------------------------------------------- exact
def _polar_like(x):
    """What five steps make of x, in 64 bits, from the steps' polynomials in the starting Gram matrix alone: each step multiplies by
    a + b S + c S^2 from the left and turns S into (a + b S + c S^2)^2 S; all these matrices commute."""
    a, b, c = COEFFICIENTS
    x = x.to(torch.float64)
    if x.shape[0] > x.shape[1]:
        return _polar_like(x.mT).mT.contiguous()
    x = x / (torch.linalg.vector_norm(x) + EPS)
    s = torch.mm(x, x.mT)
    whole = torch.eye(x.shape[0], dtype=torch.float64, device=x.device)
    for _ in range(STEPS):
        p = torch.mm(s, s).mul_(c).add_(s, alpha=b)
        p.diagonal().add_(a)
        whole = torch.mm(p, whole)
        s = torch.mm(torch.mm(p, s), p)
    return torch.mm(whole, x)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "orthogonalize":
        return [_polar_like(x) for x in s["x"]]
    if case["op"] == "step":
        weights, momentum = [], []
        for p, v in zip(s["weights"], s["momentum"]):
            g, p = p.grad.double(), p.detach().double()
            v = MOMENTUM * v.double() + g
            momentum.append(v)
            weights.append(p - LR * (DECAY * p + 0.2 * max(p.shape) ** 0.5 * _polar_like(g + MOMENTUM * v)))
        return {"weights": weights, "momentum": momentum}
    if case["op"] == "product":
        a, b = s["a"].double() * s["sa"].double()[..., None], s["b"].double() * s["sb"].double()[..., None]
        return torch.matmul(a, b.mT.contiguous())

    def values(f):
        f = f.double().movedim(-3, -1)
        unit = torch.linalg.vector_norm(f, math.inf, -1, keepdim=True)
        return torch.round(127 * f / unit).mul_(unit / 127).flatten(-3, -2)
    h, w = case["h"], case["w"]
    one, two = values(s["reference"]), values(s["target"])
    volume = torch.matmul(one, two.mT.contiguous()) / case["dim"] ** 0.5
    high, wide = -(-h // 4), -(-w // 8)
    out = volume.new_zeros(*volume.shape[:-1], high * wide * 32)
    y, x = torch.meshgrid(torch.arange(h, device="cuda"), torch.arange(w, device="cuda"), indexing="ij")
    out[..., (((y // 4) * wide + x // 8) * 32 + (y % 4) * 8 + x % 8).flatten()] = volume
    return out
