"""Newton-Schulz orthogonalisation and the Muon step (bflow_amd/muon.py, csrc/newton_schulz.hip) against plain 64-bit forms.

Tolerances (relative, Frobenius norm).  The arithmetic of a step is fp16 pairs: an operand is off by at most 2^-22 (lo is rounded at 2^-11 of a
residue of 2^-11), lo * lo is left out (2^-22), so a product of two is off by 3 * 2^-22 in the worst case, and a sum of K products in 32 bits by
another 2^-24 a term in the worst case, sqrt(K) 2^-24 as rounding goes.  A step has three products behind one another: about 9 * 2^-22 = 2e-6.
The step's map x -> a x + b x^3 + c x^5 has a slope of 3.45 at 0 and at most 3.9 on [0, 1.2]; a relative error grows only by what the map bends
(slope * x / value <= 3.9 in absolute value, near or below 1 on most of the interval), so five steps leave a few times 2e-6.  F32_TOL = 2e-5 is
ten times the error of one step.  That holds where no direction is empty.  In a matrix of rank one all others are: there the rounding of the
strong direction, 2^-22 of |X| = 1 in the worst case, is all there is, and five steps multiply it by a^5 = 3.4445^5 = 485, while the strong
direction ends at no less than 0.68 (the least of the map on the interval the steps end in): RANK_ONE_TOL = 485 * 2^-22 / 0.68 = 1.7e-4.  Results in 16 bits add their own half step: 2^-11 (fp16), 2^-8 (bf16)."""
import copy
import math

import numpy as np
import pytest
import torch

import bflow_amd
from bflow_amd import hip, muon, training
from bflow_amd.validation import DataLoading, DataSetType

DEV = "cuda:0"
F32_TOL = 2e-5
RANK_ONE_TOL = 485 * 2.0 ** -22 / 0.68
TOL = {torch.float32: F32_TOL, torch.float16: F32_TOL + 2.0 ** -11, torch.bfloat16: F32_TOL + 2.0 ** -8}
gpu = pytest.mark.gpu


def plain(x, steps=5, coefficients=muon.COEFFICIENTS, eps=1e-7):
    """The definition, in 64 bits on the CPU, on a (rows, everything else) matrix."""
    a, b, c = coefficients
    y = x.detach().cpu().double().reshape(x.shape[0], -1)
    tall = y.shape[0] > y.shape[1]
    y = y.t() if tall else y
    y = y / (y.norm() + eps)
    for _ in range(steps):
        g = y @ y.t()
        y = a * y + (b * g + c * g @ g) @ y
    return (y.t() if tall else y).reshape(x.shape)


def off(got, want):
    got, want = got.detach().cpu().double(), want.double()
    return float((got - want).norm() / want.norm())


def gradient(*shape, seed=0, size=1e-3):
    """A few strong directions, a tail of weak ones, noise."""
    rs = np.random.RandomState(seed)
    m, n = shape[0], int(np.prod(shape[1:]))
    r = max(1, min(m, n) // 4)
    x = (rs.standard_normal((m, r)) * np.logspace(0, -3, r)) @ rs.standard_normal((r, n)) + 0.03 * rs.standard_normal((m, n))
    return torch.from_numpy((size * x).astype(np.float32).reshape(shape))


# ------------------------------------------------------------------------------------------------------------------------- refusals (CPU)
def test_refuses_what_it_cannot_take():
    x = torch.zeros(4, 4)
    with pytest.raises(hip.BflowHipError, match="no CPU fallback"):
        muon.orthogonalize([x])
    with pytest.raises(hip.BflowHipError, match="list"):
        muon.orthogonalize(x)
    for bad in (0, 33, 2.5):
        with pytest.raises(hip.BflowHipError, match="steps"):
            muon.orthogonalize([], steps=bad)
    for bad in (0.0, 1e-310, 1.0, float("nan")):
        with pytest.raises(hip.BflowHipError, match="eps"):
            muon.orthogonalize([], eps=bad)
    with pytest.raises(hip.BflowHipError, match="three"):
        muon.orthogonalize([], coefficients=(1.0, 2.0))
    assert muon.orthogonalize([]) == []


def test_c_entry_refuses_bad_tables():
    """The C entry's own checks, before any launch: no GPU is touched."""
    lib = hip.lib()

    def call(rows=40, cols=80, src=256, dst=256, src_ld=80, dst_ld=80, momentum=256, steps=5, abc=muon.COEFFICIENTS, eps=1e-7, dtype=0, ws=256, ws_bytes=1 << 30, step=False):
        t = muon._table([(src, dst, momentum, src_ld, dst_ld, rows, cols)])
        if step:
            return lib.bflow_muon_step(t.ctypes.data, 1, steps, *abc, eps, 0.9, 1, 0.1, None, 0.0, ws, ws_bytes, None)
        return lib.bflow_ns_orthogonalize(t.ctypes.data, 1, dtype, steps, *abc, eps, ws, ws_bytes, None)

    for kw in (dict(rows=0), dict(cols=0), dict(cols=hip_limit() + 1), dict(rows=-1), dict(rows=1 << 16, cols=1 << 16, src_ld=1 << 16, dst_ld=1 << 16), dict(src=0), dict(dst=0),
               dict(src_ld=79), dict(dst_ld=79), dict(steps=0), dict(steps=33), dict(eps=0.0), dict(eps=1.0), dict(dtype=3), dict(dtype=-1), dict(ws=0), dict(ws=128),
               dict(ws_bytes=1024), dict(abc=(5.0, 0.0, 0.0)), dict(abc=(float("nan"), 0.0, 0.0)), dict(step=True, momentum=0)):
        assert call(**kw) == -1, kw
        assert b"newton_schulz" in lib.bflow_last_error_string() or b"ns_orthogonalize" in lib.bflow_last_error_string()
    for kw in (dict(src=0), dict(dst_ld=3), dict(step=True, momentum=0), dict(steps=0)):       # a matrix that needs no workspace is checked all the same
        assert call(rows=4, cols=8, **kw) == -1, kw
    assert lib.bflow_ns_workspace_bytes(None, 1) == -1
    empty = muon._table([])
    assert lib.bflow_ns_workspace_bytes(empty.ctypes.data, 0) == 0


def hip_limit():
    return 1 << 20


def test_optimizer_checks_its_arguments():
    w = torch.nn.Parameter(torch.zeros(4, 4))
    for kw in (dict(lr=-1.0), dict(momentum=1.0), dict(momentum=-0.1), dict(weight_decay=-1.0)):
        with pytest.raises(ValueError):
            muon.Muon([w], **kw)
    with pytest.raises(hip.BflowHipError, match="adamw=True"):
        muon.Muon([torch.nn.Parameter(torch.zeros(4))])
    with pytest.raises(hip.BflowHipError, match="adamw=True"):
        muon.Muon([torch.nn.Parameter(torch.zeros(4, 6).t())])
    with pytest.raises(hip.BflowHipError, match="float32"):
        muon.Muon([torch.nn.Parameter(torch.zeros(4, 4, dtype=torch.float16))])
    opt = muon.Muon([{"params": [w]}, {"params": [torch.nn.Parameter(torch.zeros(4))], "adamw": True}])
    with pytest.raises(hip.BflowHipError, match="adamw=True"):       # a refused group is not kept
        opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(3))]})
    assert len(opt.param_groups) == 2
    opt.step()                                                       # no gradients: nothing to do, on any device
    w.grad = torch.zeros(4, 4)
    with pytest.raises(hip.BflowHipError, match="no CPU fallback"):
        opt.step()


def test_configure_optimizers_chooses():
    from bflow_amd import configs
    m = bflow_amd.RAFTSpline(configs.model_config("E_LU4_BD2"))
    tp = dict(learning_rate=1e-4, weight_decay=1e-4, lr_scheduler=dict(use=True, total_steps=10, pct_start=0.1))
    opt, _ = training.configure_optimizers(m, tp)
    assert type(opt) is torch.optim.AdamW
    opt, sch = training.configure_optimizers(m, dict(tp, optimizer="muon", muon=dict(momentum=0.9, steps=4)))
    assert type(opt) is muon.Muon and sch is not None
    filters, rest = opt.param_groups
    assert not filters["adamw"] and rest["adamw"] and filters["momentum"] == 0.9 and filters["steps"] == 4
    assert all(p.dim() == 4 for p in filters["params"]) and all(p.dim() == 1 for p in rest["params"])
    assert len(filters["params"]) + len(rest["params"]) == len(list(m.parameters()))
    with pytest.raises(ValueError, match="optimizer"):
        training.configure_optimizers(m, dict(tp, optimizer="sgd"))


# ------------------------------------------------------------------------------------------------------------------------------- matrices
SHAPES = [(1, 1), (1, 77), (77, 1), (2, 2049), (5, 3), (63, 64), (64, 64), (64, 65), (65, 63), (128, 1152), (129, 513), (517, 131), (300, 300), (256, 567), (700, 1500)]


@gpu
@pytest.mark.parametrize("dtype", list(TOL))
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[0]}x{s[1]}")
def test_one_matrix(shape, dtype):
    x = gradient(*shape, seed=sum(shape)).to(dtype)
    before = x.clone()
    dev = x.to(DEV)
    (y,) = muon.orthogonalize([dev])
    assert y.shape == x.shape and y.dtype == dtype and y.is_contiguous()
    assert off(y, plain(x)) < TOL[dtype]
    assert torch.equal(dev.cpu(), before)


@gpu
@pytest.mark.parametrize("steps", [1, 2, 3, 6])
def test_steps_and_coefficients(steps):
    x = gradient(96, 200, seed=steps)
    for abc in (muon.COEFFICIENTS, (1.5, -0.5, 0.0), (1.875, -1.25, 0.375)):
        (y,) = muon.orthogonalize([x.to(DEV)], steps=steps, coefficients=abc)
        assert off(y, plain(x, steps, abc)) < F32_TOL


@gpu
def test_a_list_equals_its_plain_forms_and_repeats_bit_for_bit():
    """More matrices than one round of launches takes, types mixed, filters among them, an empty one: each right, in order, and the same bits twice."""
    shapes = [(1 + 7 * k % 130, 1 + 13 * k % 90) for k in range(75)] + [(64, 5, 7, 7), (96, 64, 1, 1), (4, 256, 3, 3)]
    kinds = list(TOL)
    xs = [gradient(*s, seed=k).to(kinds[k % 3] if k < 70 else torch.float32) for k, s in enumerate(shapes)]
    xs.insert(3, torch.zeros(0, 5))
    xs.insert(9, torch.zeros(5, 0))
    dev = [x.to(DEV) for x in xs]
    ys, again = muon.orthogonalize(dev), muon.orthogonalize(dev)
    for x, y, z in zip(xs, ys, again):
        assert y.shape == x.shape and torch.equal(y, z)
        if x.numel():
            assert off(y, plain(x)) < TOL[x.dtype]


@gpu
def test_strides():
    """Rows further apart than they are long, a transposed view, a slice that starts at an odd element."""
    big = gradient(150, 401, seed=1)
    dev = big.to(DEV)
    cases = [(dev[:70, :100], big[:70, :100]), (dev[3:90, 7:], big[3:90, 7:]), (dev.t(), big.t()), (dev[::2, 1:60], big[::2, 1:60]), (dev[:1, 5:9], big[:1, 5:9]),
             (dev[:, ::3], big[:, ::3]), (dev[0].expand(6, 401), big[0].expand(6, 401))]
    ys = muon.orthogonalize([d for d, _ in cases])
    for y, (_, x) in zip(ys, cases):
        assert y.is_contiguous() and off(y, plain(x)) < F32_TOL


@gpu
def test_zero_tiny_huge_and_lost_values():
    x = gradient(40, 100, seed=2)
    nan, inf, rank1 = x.clone(), x.clone(), torch.outer(x[:, 0], x[0])
    nan[3, 5], inf[39, 99] = float("nan"), float("-inf")
    zero, tiny, huge = torch.zeros(33, 70), x * 1e-30, x * 1e30
    one_row = torch.zeros(40, 100)
    one_row[17] = x[17]
    ys = muon.orthogonalize([t.to(DEV) for t in (zero, tiny, huge, nan, inf, rank1, one_row)])
    assert not ys[0].any()
    assert off(ys[1], plain(tiny)) < F32_TOL and off(ys[2], plain(huge)) < F32_TOL
    assert torch.isnan(ys[3]).all() and torch.isnan(ys[4]).all()
    assert off(ys[5], plain(rank1)) < RANK_ONE_TOL and off(ys[6], plain(one_row)) < F32_TOL      # (one row: the others hold no rounding either)
    assert not ys[6][:17].any() and not ys[6][18:].any()


@gpu
@pytest.mark.parametrize("eps", [1e-60, 1e-300])
def test_eps_below_32_bits(eps):
    """eps only has to keep zero matrices apart from 0 / 0, and may be smaller than a 32-bit number."""
    xs = [gradient(40, 100, seed=1), gradient(300, 280, seed=2), gradient(6, 40, seed=3), torch.zeros(40, 100), torch.zeros(300, 280), torch.zeros(6, 40)]
    for group in (xs, xs[:1] + xs[3:4]):
        for x, y in zip(group, muon.orthogonalize([x.to(DEV) for x in group], eps=eps)):
            assert off(y, plain(x, eps=eps)) < F32_TOL if x.any() else not y.any()


@gpu
@pytest.mark.parametrize("dtype", list(TOL))
def test_small_matrices_around_the_limits_of_their_kernel(dtype):
    """Few rows, up to the sizes where the kernel in one workgroup ends and just beyond, wide and tall, alone and beside larger ones.  Held in 64 bits
    below the limits: there fp32 results are off by their own rounding alone."""
    shapes = [(r, c) for r in (1, 2, 4, 5, 8) for c in (1, 8, 513, 2049)] + [(r, c) for r in (9, 15, 16, 17, 31, 32) for c in (9, 33, 129, 256)]
    shapes += [(8, 16384), (8, 16385), (1, 131072), (1, 131073), (32, 257), (33, 40), (16, 512), (16, 513), (9, 910), (9, 911), (3, 3), (2, 70001)]
    shapes += [(c, r) for r, c in shapes if c != r]
    xs = [gradient(*s, seed=k).to(dtype) for k, s in enumerate(shapes)]
    dev = [x.to(DEV) for x in xs]
    alone = muon.orthogonalize(dev)
    beside = muon.orthogonalize([torch.ones(200, 300, device=DEV, dtype=dtype)] + dev)[1:]
    for x, y, z in zip(xs, alone, beside):
        r, numbers = min(x.shape), x.numel()
        held = r <= 32 and numbers <= (1 << 17 if r <= 8 else 1 << 13)
        # 64 bits: 2^-24 for the result's rounding; five steps of 2^-53 * sqrt(131072) each, at a growth of 485, stay far below it
        limit = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11 + 2.0 ** -24, torch.bfloat16: 2.0 ** -8 + 2.0 ** -24}[dtype] * 1.001 if held else TOL[dtype]
        if dtype is torch.float16:
            limit += 2.0 ** -25 * math.sqrt(numbers) / float(plain(x).norm())           # below 2^-14 its step is 2^-24 whatever the value
        assert off(y, plain(x)) < limit, (tuple(x.shape), limit)
        assert not held or torch.equal(y, z)


@gpu
@pytest.mark.parametrize("dtype", list(TOL))
def test_result_over_the_matrix_itself(dtype):
    """The C entry with dst = src: small matrices, panels and larger ones; the same bits as into another place."""
    for shapes in ([(7, 90), (30, 100), (100, 20), (5, 3000), (64, 576)], [(300, 280), (12, 40)], [(32, 245), (500, 16), (33, 33), (20, 400), (2, 40000)]):
        xs = [gradient(*s, seed=k).to(dtype).to(DEV) for k, s in enumerate(shapes)]
        want = muon.orthogonalize(xs)
        table = muon._table([(x.data_ptr(), x.data_ptr(), 0, x.shape[1], x.shape[1], *x.shape) for x in xs])
        hip.ns_orthogonalize(table, dtype, xs[0].device, 5, muon.COEFFICIENTS, 1e-7)
        assert all(torch.equal(x, y) for x, y in zip(xs, want))


@gpu
def test_small_matrices_lost_values_and_steps():
    x = gradient(12, 90, seed=4)
    nan, inf, zero, small, large = x.clone(), x.clone(), torch.zeros(8, 3), x * 1e-37, x * 1e37
    nan[11, 89], inf[0, 0] = float("nan"), float("inf")
    ys = muon.orthogonalize([t.to(DEV) for t in (nan, inf, zero, small, large)])
    assert torch.isnan(ys[0]).all() and torch.isnan(ys[1]).all() and not ys[2].any()
    assert off(ys[3], plain(small)) < 2.0 ** -23 and off(ys[4], plain(large)) < 2.0 ** -23
    for steps, eps in ((1, 1e-7), (2, 0.5), (9, 1e-7)):
        for abc in (muon.COEFFICIENTS, (1.5, -0.5, 0.0)):
            for shape in ((12, 90), (30, 31), (3, 1200)):
                x = gradient(*shape, seed=steps)
                (y,) = muon.orthogonalize([x.to(DEV)], steps=steps, coefficients=abc, eps=eps)
                assert off(y, plain(x, steps, abc, eps)) < 2.0 ** -23, (steps, eps, abc, shape)


@gpu
def test_refuses_on_the_device():
    x = torch.zeros(4, 4, device=DEV)
    with pytest.raises(hip.BflowHipError, match="two dimensions"):
        muon.orthogonalize([x[0]])
    with pytest.raises(hip.BflowHipError, match="dtype"):
        muon.orthogonalize([x.double()])
    with pytest.raises(hip.BflowHipError, match="coefficients"):
        muon.orthogonalize([x], coefficients=(5.0, 0.0, 0.0))


@gpu
def test_on_another_stream_and_in_a_graph():
    """Two streams at once (a workspace each), then a captured call: replays follow the input, also between eager calls of other lists."""
    xs = [gradient(64, 576, seed=1), gradient(256, 567, seed=2), gradient(300, 40, seed=3)]
    a, b = [x.to(DEV) for x in xs], [(2 * x.flip(1)).to(DEV) for x in xs]
    want_a, want_b = muon.orthogonalize(a), muon.orthogonalize(b)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s1):
        ya = [muon.orthogonalize(a) for _ in range(3)]
    with torch.cuda.stream(s2):
        yb = [muon.orthogonalize(b) for _ in range(3)]
    torch.cuda.synchronize()
    for got, want in ((ya, want_a), (yb, want_b)):
        for y in got:
            assert all(torch.equal(p, q) for p, q in zip(y, want))
    static = [x.clone() for x in a]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = muon.orthogonalize(static)
    for source, want in ((a, want_a), (b, want_b), (a, want_a)):
        for s, x in zip(static, source):
            s.copy_(x)
        graph.replay()
        muon.orthogonalize([x.to(DEV) for x in xs[:2]])
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shapes", [[(2900, 2950)], [(1000, 1020)] * 8, [(70, 3000)] + [(1000, 1020)] * 8,
                                    [(1000, 4000)] + [(1000, 1020)] * 4 + [(4000, 1000), (1000, 900)]], ids=["one", "eight", "nine", "lengths"])
def test_last_tiles_cut_along_the_contraction(shapes, dtype):
    """276, 288 and 289 tiles of 128 x 128: those behind the 256th are cut; tiles of two lengths: the long ones are.  Against 64 bits on the device, in front of and behind other calls; twice the same
    bits; and through a step."""
    xs = [gradient(*s, seed=k).to(dtype).to(DEV) for k, s in enumerate(shapes)]

    def exact(x):
        a, b, c = muon.COEFFICIENTS
        tall = x.shape[0] > x.shape[1]
        y = x.double() / (x.double().norm() + 1e-7)
        y = y.t().contiguous() if tall else y
        for _ in range(5):
            g = y @ y.t()
            y = a * y + (b * g + c * g @ g) @ y
        return y.t() if tall else y
    ys = muon.orthogonalize(xs)
    muon.orthogonalize([xs[-1][:300, :310]])
    assert all(torch.equal(y, z) for y, z in zip(ys, muon.orthogonalize(xs)))
    for x, y in zip(xs, ys):
        assert off(y, exact(x).cpu()) < TOL[dtype]
    if dtype is torch.float32:
        ps = [torch.nn.Parameter(torch.zeros_like(x)) for x in xs]
        for p, x in zip(ps, xs):
            p.grad = x
        muon.Muon(ps, lr=0.5, momentum=0.0).step()
        for p, y in zip(ps, ys):
            assert off(p, y.cpu() * (-0.1 * math.sqrt(max(y.shape)))) < 2.0 ** -22


@gpu
@pytest.mark.parametrize("shape,dtype", [((1024, 1 << 20), torch.bfloat16), ((1 << 20, 200), torch.float32), ((8192, 100), torch.float16)], ids=["wide", "tall", "panels"])
def test_longest_rows(shape, dtype):
    """Byte offsets behind 2^32 in the workspace, 2^20 columns or rows, against 64 bits on the device: slices of the result, from the Gram matrix."""
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(shape, generator=g, device=DEV).to(dtype)
    tall = shape[0] > shape[1]
    (y,) = muon.orthogonalize([x])
    wide, out = (x.t(), y.t()) if tall else (x, y)
    S = torch.zeros(wide.shape[0], wide.shape[0], dtype=torch.float64, device=DEV)
    for c in range(0, wide.shape[1], 1 << 16):
        part = wide[:, c:c + (1 << 16)].double()
        S += part @ part.t()
    # every step is a polynomial of S; all singular values of these matrices are within a factor of two
    norm, Q, eye = S.trace().sqrt() + 1e-7, None, torch.eye(S.shape[0], dtype=torch.float64, device=DEV)
    S = S / norm ** 2
    for _ in range(5):
        a, b, c = muon.COEFFICIENTS
        P = a * eye + b * S + c * S @ S
        Q, S = P if Q is None else P @ Q, P @ S @ P
    for c in (0, wide.shape[1] // 2 + 57, wide.shape[1] - 300):
        want = (Q @ wide[:, c:c + 300].double() / norm).cpu()
        assert off(out[:, c:c + 300], want) < TOL[dtype]
    del x, y, wide, out
    torch.cuda.empty_cache()


# ------------------------------------------------------------------------------------------------------------------------------- the step
def plain_step(p, g, v, lr, decay, mu, nesterov, **kw):
    p, g, v = (t.detach().cpu().double() for t in (p, g, v))
    v = mu * v + g
    m, n = p.shape[0], p[0].numel()
    return p * (1 - lr * decay) - lr * 0.2 * math.sqrt(max(m, n)) * plain(g + mu * v if nesterov else v, **kw), v


@gpu
@pytest.mark.parametrize("nesterov,mu,decay", [(True, 0.95, 0.1), (False, 0.9, 0.0), (True, 0.0, 0.01)])
def test_steps_of_the_optimizer(nesterov, mu, decay):
    """Three steps on filters, matrices, tall and wide; the update itself is held to the tolerance, not only the weights."""
    shapes = [(64, 5, 7, 7), (4, 256, 3, 3), (96, 64, 1, 1), (576, 256), (1, 9), (130, 70)]
    lr = 0.02
    ps = [torch.nn.Parameter(gradient(*s, seed=k, size=1.0).to(DEV)) for k, s in enumerate(shapes)]
    frozen = torch.nn.Parameter(torch.ones(3, 3, device=DEV))
    opt = muon.Muon(ps + [frozen], lr=lr, momentum=mu, weight_decay=decay, nesterov=nesterov)
    vs = [torch.zeros(p.shape, dtype=torch.float64) for p in ps]
    for t in range(3):
        before = [p.detach().clone() for p in ps]
        versions = [p._version for p in ps]
        for k, p in enumerate(ps):
            p.grad = gradient(*shapes[k], seed=10 * t + k).to(DEV)
        opt.step()
        for k, p in enumerate(ps):
            want, vs[k] = plain_step(before[k], p.grad, vs[k], lr, decay, mu, nesterov)
            v = opt.state[p]["momentum_buffer"]
            assert off(v, vs[k]) < 2.0 ** -22                       # a rounding for each step, 2^-24 each
            moved, wanted = p.detach().cpu().double() - before[k].cpu().double(), want - before[k].cpu().double()
            # weights are stored in 32 bits: 2^-24 of a weight on top of the update's own error (momentum: 3 * 2^-24, inside it)
            assert float((moved - wanted).norm()) < F32_TOL * float(wanted.norm()) + 2.0 ** -23 * float(want.norm())
            assert p._version > versions[k]
            vs[k] = v.cpu().double()
    assert torch.equal(frozen, torch.ones_like(frozen)) and frozen not in opt.state


@gpu
def test_optimizer_takes_strided_gradients_and_a_rate_on_the_device():
    p = torch.nn.Parameter(gradient(64, 96, 3, 3, seed=1, size=1.0).to(DEV))
    q = torch.nn.Parameter(p.detach().clone())
    g = gradient(64, 96, 3, 3, seed=2).to(DEV)
    p.grad, q.grad = g, g.to(memory_format=torch.channels_last)
    rate = torch.tensor(0.5, device=DEV)
    a, b = muon.Muon([p], lr=0.02), muon.Muon([q], lr=rate)
    a.step()
    rate.fill_(0.02)
    b.zero_grad(set_to_none=False)
    q.grad = g.to(memory_format=torch.channels_last)
    q.data.copy_(gradient(64, 96, 3, 3, seed=1, size=1.0))
    b.step()
    assert torch.equal(p, q)
    b.load_state_dict(copy.deepcopy(a.state_dict()))
    assert torch.equal(b.state[q]["momentum_buffer"], a.state[p]["momentum_buffer"])


@gpu
@pytest.mark.parametrize("shapes", [[(2, 64, 3, 3), (2, 128, 1, 1), (8, 1, 1, 1), (20, 17), (32, 31), (1, 5), (70, 4, 2, 1), (200, 16)],
                                    [(2, 64, 3, 3), (20, 17), (64, 5, 7, 7), (40, 8, 3, 3), (96, 64, 1, 1)]], ids=["alone", "beside"])
def test_small_filters_step(shapes):
    """Heads and first layers, as the step's kernel for small matrices takes them, with a rate on the device, eager and captured."""
    rate = torch.tensor(0.02, device=DEV)

    def make():
        return [torch.nn.Parameter(gradient(*s, seed=k, size=1.0).to(DEV)) for k, s in enumerate(shapes)]
    ps, qs = make(), make()
    a = muon.Muon(ps, lr=0.02, weight_decay=0.1)
    b = muon.Muon(qs, lr=rate, weight_decay=0.1, capturable=True)
    grads = [torch.empty(s, device=DEV) for s in shapes]
    for p, q, g in zip(ps, qs, grads):
        p.grad = q.grad = g
    vs, graph = [torch.zeros(s, dtype=torch.float64) for s in shapes], torch.cuda.CUDAGraph()
    for t in range(4):
        for k, g in enumerate(grads):
            g.copy_(gradient(*shapes[k], seed=10 * t + k))
        before = [p.detach().cpu().clone() for p in ps]
        a.step()
        if t == 0:
            b.step()
            torch.cuda.synchronize()
            with torch.cuda.graph(graph):
                b.step()
        else:
            graph.replay()
        for k, p in enumerate(ps):
            want, vs[k] = plain_step(before[k], grads[k], vs[k], 0.02, 0.1, 0.95, True)
            moved, wanted = p.detach().cpu().double() - before[k].double(), want - before[k].double()
            assert float((moved - wanted).norm()) < F32_TOL * float(wanted.norm()) + 2.0 ** -23 * float(want.norm())
            assert torch.equal(p, qs[k])
            vs[k] = a.state[p]["momentum_buffer"].cpu().double()


@gpu
def test_a_capture_needs_states_and_says_so(monkeypatch):
    w, x = torch.nn.Parameter(torch.ones(4, 4, device=DEV)), torch.nn.Parameter(torch.ones(4, device=DEV))
    w.grad, x.grad = torch.ones(4, 4, device=DEV), torch.ones(4, device=DEV)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    groups = lambda: [{"params": [w]}, {"params": [x], "adamw": True}]
    with pytest.raises(hip.BflowHipError, match="capturable"):
        muon.Muon(groups()).step()
    for group in groups():
        with pytest.raises(hip.BflowHipError, match="first step"):
            muon.Muon([group], capturable=True).step()
    for lr in (torch.ones(2, device=DEV), torch.ones((), device=DEV, dtype=torch.float64), torch.ones(0, device=DEV)):
        monkeypatch.undo()
        with pytest.raises(hip.BflowHipError, match="float32 scalar"):
            muon.Muon([w], lr=lr).step()
    assert torch.equal(w, torch.ones_like(w)) and torch.equal(x, torch.ones_like(x))


@gpu
def test_adamw_group_is_adamw():
    w, x = torch.nn.Parameter(torch.randn(7, 5, device=DEV)), torch.nn.Parameter(torch.randn(9, device=DEV))
    y = torch.nn.Parameter(x.detach().clone())
    opt = muon.Muon([{"params": [w]}, {"params": [x], "adamw": True}], lr=0.01, weight_decay=0.1)
    ref = torch.optim.AdamW([y], lr=0.01, weight_decay=0.1)
    for t in range(3):
        w.grad = torch.randn(7, 5, device=DEV)
        x.grad = torch.randn(9, device=DEV)
        y.grad = x.grad.clone()
        opt.step()
        ref.step()
        assert torch.equal(x, y)


@gpu
def test_training_steps_with_muon_eager_and_graphed():
    """configure_optimizers(optimizer: muon) through the whole training step, eager against one captured graph; a plain update beside it."""
    from bflow_amd import configs, synthetic
    from bflow_amd.weights import deterministic_state_dict
    cfg = configs.model_config("E_LU4_BD2")
    B, H, W = 1, 64, 96
    tp = dict(learning_rate=2e-4, weight_decay=1e-4, optimizer="muon", lr_scheduler=dict(use=True, total_steps=50, pct_start=0.3))

    def batch(seed):
        rs = np.random.RandomState(seed)
        to = lambda a: torch.from_numpy(a).to(DEV)
        return {DataLoading.EV_REPR: to(synthetic.voxel_grid(B, 9, H, W, seed=seed)), DataLoading.FLOW: to(rs.standard_normal((B, 2, H, W)).astype(np.float32) * 4),
                DataLoading.FLOW_VALID: to(rs.rand(B, H, W) > 0.2), DataLoading.DATASET_TYPE: [DataSetType.DSEC] * B}

    def make(capturable):
        m = bflow_amd.RAFTSpline(cfg)
        m.load_state_dict(deterministic_state_dict(m, seed=0))
        m.to(DEV).train()
        opt, sch = training.configure_optimizers(m, tp, capturable=capturable)
        return m, opt, sch, training.TrainStep(m, num_iter_train=2)

    batches = [batch(5), batch(6), batch(7)]
    m1, opt1, sch1, step1 = make(False)
    eager = []
    for k, b in enumerate(batches):
        opt1.zero_grad(set_to_none=True)
        out = step1(b)
        out["loss"].backward()
        if k == 0:
            p = m1.update_block.gru.convz1.weight
            before, lr = p.detach().clone(), opt1.param_groups[0]["lr"]
            want, _ = plain_step(before, p.grad, torch.zeros_like(p), lr, 1e-4, 0.95, True)
        opt1.step()
        if k == 0:
            moved, wanted = p.detach().cpu().double() - before.cpu().double(), want - before.cpu().double()
            assert float((moved - wanted).norm()) < F32_TOL * float(wanted.norm()) + 2.0 ** -23 * float(want.norm())
        sch1.step()
        eager.append(float(out["loss"].detach()))
    m2, opt2, sch2, step2 = make(True)
    gstep = training.GraphedTrainStep(step2, opt2, sch2)
    graphed = [float(gstep(b)["loss"].detach()) for b in batches]
    # the same kernels on the same numbers, but for the order of the look-up adjoint's sums (2^-24 each, through three updates)
    assert graphed == pytest.approx(eager, rel=1e-3)
    assert all(bool(torch.isfinite(p).all()) for p in m2.parameters())


# ------------------------------------------------------------------------------------------------------------ the other sets of tiles
@gpu
@pytest.mark.parametrize("dtype", list(TOL))
@pytest.mark.parametrize("shapes", [[(390 + k % 11, 385 + 3 * k % 40) for k in range(20)],         # 560 blocks of 64 x 64 in the Gram matrices: large tiles
                                    [(257, 300), (40, 1000), (1, 5), (300, 257)],                   # one matrix over 256 rows: small tiles for all
                                    [(256, 256), (193, 2000), (64, 64), (1, 3000), (2500, 65), (130, 129)]],     # at most 256 rows: panels
                         ids=["large", "small", "panels"])
def test_lists_of_every_set(shapes, dtype):
    xs = [gradient(*s, seed=k).to(dtype) for k, s in enumerate(shapes)]
    ys = muon.orthogonalize([x.to(DEV) for x in xs])
    for x, y in zip(xs, ys):
        assert off(y, plain(x)) < TOL[dtype]


@gpu
@pytest.mark.parametrize("shapes", [[(390, 385 + k) for k in range(20)], [(300, 280), (7, 9)], [(128, 1920), (192, 500), (256, 80), (9, 200)]], ids=["large", "small", "panels"])
def test_step_of_every_set(shapes):
    ps = [torch.nn.Parameter(gradient(*s, seed=k, size=1.0).to(DEV)) for k, s in enumerate(shapes)]
    opt = muon.Muon(ps, lr=0.05, weight_decay=0.1)
    before = [p.detach().clone() for p in ps]
    for k, p in enumerate(ps):
        p.grad = gradient(*shapes[k], seed=50 + k).to(DEV)
    opt.step()
    for p, old in zip(ps, before):
        want, v = plain_step(old, p.grad, torch.zeros_like(old), 0.05, 0.1, 0.95, True)
        moved, wanted = p.detach().cpu().double() - old.cpu().double(), want - old.cpu().double()
        assert float((moved - wanted).norm()) < F32_TOL * float(wanted.norm()) + 2.0 ** -23 * float(want.norm())
        assert off(opt.state[p]["momentum_buffer"], v) < 2.0 ** -23


@gpu
def test_long_matrices():
    """Many panels of a workgroup, many parts of a Gram matrix; columns that end inside a panel."""
    for shape in ((3, 70001), (64, 20033), (200, 9001), (70001, 2)):
        x = gradient(*shape, seed=shape[0])
        (y,) = muon.orthogonalize([x.to(DEV)])
        assert off(y, plain(x)) < F32_TOL


@gpu
def test_results_of_one_type_share_a_buffer_and_stay_apart():
    xs = [gradient(3, 5, seed=k).to(DEV) for k in range(4)]
    ys = muon.orthogonalize(xs)
    keep = [y.clone() for y in ys]
    ys[1].fill_(7.0)
    assert torch.equal(ys[0], keep[0]) and torch.equal(ys[2], keep[2]) and all(y.data_ptr() % 256 == 0 for y in ys)


# ------------------------------------------------------------------------------------------------------------ results rounded once
def spectrum(kind, m, n, seed):
    """Matrices whose singular values are no gradient's: all alike, a Gaussian's, one alone, a few and no others."""
    rs = np.random.RandomState(seed)
    if kind == "orthogonal":
        q = torch.linalg.qr(torch.from_numpy(rs.standard_normal((max(m, n), min(m, n)))))[0]
        return q if m >= n else q.t().contiguous()
    if kind == "gaussian":
        return torch.from_numpy(rs.standard_normal((m, n)))
    if kind == "constant":
        return torch.full((m, n), 0.75, dtype=torch.float64)
    return torch.from_numpy(np.round(rs.standard_normal((m, 3)) * 4) @ np.round(rs.standard_normal((3, n)) * 4))      # "rank three": whole numbers, most below 256


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kind", ["orthogonal", "gaussian", "constant", "rank three"])
def test_16_bit_results_are_those_of_32_bits_rounded(kind, dtype):
    """An entry of the result is a 32-bit-class number z, next to the exact x, rounded once.  A number's distance from the nearest 16-bit number changes by no
    more than the number itself does, so |y - x| <= |z - rounded(z)| + |z - x| <= |x - rounded(x)| + 2 |z - x|, whatever the spectrum; |z - x| is held as in
    32 bits (few directions: as the rank-one matrices above).  Panels, and both sets of tiles of the products."""
    for k, shapes in enumerate(([(200, 230)], [(300, 300)], [(400, 500), (500, 400)], [(390 + j, 385 + 3 * j) for j in range(20)])):
        xs = [spectrum(kind, *s, seed=7 * k + j).to(dtype) for j, s in enumerate(shapes)]
        for x, y in zip(xs, muon.orthogonalize([x.to(DEV) for x in xs])):
            want = plain(x)
            few = kind in ("constant", "rank three")
            assert off(y, want) < off(want.to(dtype), want) + 2 * (RANK_ONE_TOL if few else F32_TOL), tuple(x.shape)


@gpu
@pytest.mark.parametrize("shapes", [[(4, 2304), (7, 1500)], [(16, 512)], [(32, 256)], [(64, 576), (576, 64), (128, 300)], [(300, 281)], [(300, 280), (280, 300)],
                                    [(390, 388 + 4 * k) for k in range(20)]], ids=["4 and 8 rows", "16 rows", "32 rows", "panels", "products", "products by fours", "large tiles"])
def test_decay_below_half_a_step_of_the_weights(shapes):
    """lr = decay = 1e-4, as the training configuration has it: 1e-8 of a weight, a sixth of half its step.  It is lost on any one weight, not on all: along p,
    p' - (p - rate X) is -lr decay p plus the weights' roundings, each uniform over at most 2^-24 |p| to either side and independent of p beside an update
    of many steps.  Their share is sqrt(sum p^4) / sum p^2 * 2^-24 / sqrt(3), 2^-24 / sqrt(n) for Gaussian weights; X's own error, F32_TOL of an update of
    2e-5 against weights of 0.04, lies across p but for 1 / sqrt(n) of it: 1e-8 / sqrt(n).  Six times the two together, below half of what is looked for."""
    lr = decay = 1e-4
    ps = [torch.nn.Parameter((0.04 * torch.randn(s, generator=torch.Generator().manual_seed(k))).to(DEV)) for k, s in enumerate(shapes)]
    before = [p.detach().cpu().double() for p in ps]
    for k, p in enumerate(ps):
        p.grad = gradient(*shapes[k], seed=30 + k).to(DEV)
    rate = torch.tensor(lr, device=DEV) if len(shapes) == 1 else lr
    muon.Muon(ps, lr=rate, weight_decay=decay, momentum=0.0).step()
    moved = total = n = 0
    for p, old in zip(ps, before):
        left = p.detach().cpu().double() - (old - lr * 0.2 * math.sqrt(max(p.shape)) * plain(p.grad))
        moved, total, n = moved + float((left * old).sum()), total + float((old * old).sum()), n + old.numel()
    tolerance = 6 * (2.0 ** -24 + 1e-8) / math.sqrt(n)
    assert tolerance < 0.5 * lr * decay and abs(moved / total + lr * decay) < tolerance, moved / total


@gpu
@pytest.mark.parametrize("decay", [0.0, 0.1])
def test_lost_weights_stay_alone(decay):
    """An infinite weight stays infinite and a NaN stays one, with and without decay; their neighbours do not see them.  A matrix of each kernel."""
    for shape in ((6, 300), (20, 40), (64, 577), (300, 280), (280, 299)):
        p = torch.nn.Parameter(gradient(*shape, seed=1, size=1.0).to(DEV))
        q = torch.nn.Parameter(p.detach().clone())
        with torch.no_grad():
            p[0, 0], p[1, 2], p[5, 39] = float("inf"), float("-inf"), float("nan")
        p.grad = q.grad = gradient(*shape, seed=2).to(DEV)
        muon.Muon([p, q], lr=0.1, weight_decay=decay).step()
        assert p[0, 0] == float("inf") and p[1, 2] == float("-inf") and torch.isnan(p[5, 39])
        with torch.no_grad():
            p[0, 0], p[1, 2], p[5, 39] = q[0, 0], q[1, 2], q[5, 39]
        assert torch.equal(p, q)


def test_matrices_beyond_the_kernels_are_refused_early():
    """Where a parameter is given to the optimiser, not in its first step, and with the same error whatever the size."""
    long, many = torch.nn.Parameter(torch.zeros((1 << 20) + 1, 1)), torch.nn.Parameter(torch.empty(1 << 16, (1 << 14) + 1, device="meta"))
    for p in (long, many, torch.nn.Parameter(torch.empty(1 << 33, 2, device="meta")), torch.nn.Parameter(torch.empty(4, 1 << 11, 1 << 10, device="meta"))):
        with pytest.raises(hip.BflowHipError, match="at most"):
            muon.Muon([p])
        assert muon.Muon([{"params": [p], "adamw": True}])
    assert muon.Muon([torch.nn.Parameter(torch.empty(1 << 20, 1 << 10, device="meta"))])


@gpu
def test_orthogonalize_refuses_what_is_too_large():
    one = torch.zeros(1, 1, device=DEV)
    for shape in (((1 << 20) + 1, 2), (2, (1 << 32) + 7), (1 << 16, 1 << 16), (1 << 40, 1)):
        with pytest.raises(hip.BflowHipError, match="matrix 1: .*at most"):
            muon.orthogonalize([one, one.expand(shape)])


@gpu
def test_results_are_tensors_of_their_own():
    """Writing into one result neither bumps the version of another that a graph has saved nor touches it; each holds its own storage."""
    xs = [gradient(30, 50, seed=k).to(DEV) for k in range(3)] + [gradient(300, 20, seed=4).to(DEV), gradient(2, 3, seed=5).to(DEV)]
    ys = muon.orthogonalize(xs)
    w = torch.ones(30, 50, device=DEV, requires_grad=True)
    loss = (w * ys[0]).sum()
    keep = [y.clone() for y in ys]
    for y in ys[1:]:
        y.fill_(7.0)
    loss.backward()
    assert torch.equal(w.grad, keep[0]) and torch.equal(ys[0], keep[0])
    for y, x in zip(ys, xs):
        assert y._base is None and y.storage_offset() == 0 and y.untyped_storage().nbytes() == 4 * x.numel()
    assert len({y.untyped_storage().data_ptr() for y in ys}) == len(ys)


@gpu
def test_the_recorded_step_moves_every_filter_as_the_formula_says():
    """Three replays of a captured training step: each moves every filter by the plain step of its own gradient, at the scheduled rate, from the momentum of the
    step before (none in front of the first: warm-up steps leave nothing behind).  Beside it the eager step from the same start: all filters' movements
    together.  Gradients of the two differ by the order of the look-up adjoint's sums, 1e-5 of a filter's gradient at most; that is multiplied by 485 / 0.68
    where it is all that a direction holds: 7e-3 a step, 2e-2 in three.  A rate that did not follow the schedule would show as 0.35."""
    from bflow_amd import configs, synthetic
    from bflow_amd.weights import deterministic_state_dict
    B, H, W = 1, 64, 96
    tp = dict(learning_rate=2e-4, weight_decay=1e-4, optimizer="muon", lr_scheduler=dict(use=True, total_steps=50, pct_start=0.3))

    def batch(seed):
        rs = np.random.RandomState(seed)
        to = lambda a: torch.from_numpy(a).to(DEV)
        return {DataLoading.EV_REPR: to(synthetic.voxel_grid(B, 9, H, W, seed=seed)), DataLoading.FLOW: to(rs.standard_normal((B, 2, H, W)).astype(np.float32) * 4),
                DataLoading.FLOW_VALID: to(rs.rand(B, H, W) > 0.2), DataLoading.DATASET_TYPE: [DataSetType.DSEC] * B}

    def make(capturable):
        m = bflow_amd.RAFTSpline(configs.model_config("E_LU4_BD2"))
        m.load_state_dict(deterministic_state_dict(m, seed=0))
        m.to(DEV).train()
        return (m,) + tuple(training.configure_optimizers(m, tp, capturable=capturable))

    batches = [batch(5), batch(6), batch(7)]
    m1, opt1, sch1 = make(False)
    start = [p.detach().cpu().double() for p in opt1.param_groups[0]["params"]]
    step1 = training.TrainStep(m1, num_iter_train=2)
    for b in batches:
        opt1.zero_grad(set_to_none=True)
        step1(b)["loss"].backward()
        opt1.step()
        sch1.step()
    opt1.zero_grad(set_to_none=True)

    m2, opt2, sch2 = make(True)
    gstep = training.GraphedTrainStep(training.TrainStep(m2, num_iter_train=2), opt2, sch2)
    filters, rest = (g["params"] for g in opt2.param_groups)
    rates, vs, moments = [], [torch.zeros(p.shape, dtype=torch.float64) for p in filters], [torch.zeros(p.shape, dtype=torch.float64) for p in rest]
    for n, b in enumerate(batches):
        before = [p.detach().cpu().double() for p in filters]
        rates.append(float(opt2.param_groups[0]["lr"]))
        gstep(b)
        torch.cuda.synchronize()
        for k, p in enumerate(filters):
            assert bool(p.grad.any())
            want, vs[k] = plain_step(before[k], p.grad, vs[k], rates[-1], 1e-4, 0.95, True)
            v = opt2.state[p]["momentum_buffer"].cpu().double()
            assert off(v, vs[k]) < 2.0 ** -22
            moved, wanted = p.detach().cpu().double() - before[k], want - before[k]
            assert float((moved - wanted).norm()) < F32_TOL * float(wanted.norm()) + 2.0 ** -23 * float(want.norm())
            vs[k] = v
        for k, p in enumerate(rest):
            state = opt2.state[p]
            want = 0.9 * moments[k] + 0.1 * p.grad.cpu().double()
            assert float(state["step"]) == n + 1
            moments[k] = state["exp_avg"].cpu().double()
            assert float((moments[k] - want).norm()) <= 2.0 ** -22 * (float(want.norm()) + float(p.grad.norm()))
    assert 0 < rates[0] < rates[1] < rates[2]
    apart = total = 0.0
    for p, q, s in zip(opt1.param_groups[0]["params"], filters, start):
        moved = p.detach().cpu().double() - s
        assert bool(moved.any())
        apart, total = apart + float((q.detach().cpu().double() - s - moved).norm()) ** 2, total + float(moved.norm()) ** 2
    assert apart < (2e-2) ** 2 * total, math.sqrt(apart / total)


def test_a_groups_own_numbers_are_checked():
    """What a group sets for itself is held to what the optimiser's defaults are held to: two and a half steps are not two."""
    make = lambda: torch.nn.Parameter(torch.zeros(4, 4))
    opt = muon.Muon([{"params": [make()], "momentum": 0.5, "steps": 3}])
    for kw, error in ((dict(steps=2.5), hip.BflowHipError), (dict(steps=0), hip.BflowHipError), (dict(eps=0.0), hip.BflowHipError), (dict(coefficients=(1.0,)), hip.BflowHipError),
                      (dict(momentum=1.0), ValueError), (dict(weight_decay=-0.1), ValueError), (dict(lr=float("nan")), ValueError)):
        with pytest.raises(error):
            opt.add_param_group({"params": [make()], **kw})
        with pytest.raises(error):
            muon.Muon([{"params": [make()], **kw}])
    assert len(opt.param_groups) == 1 and opt.param_groups[0]["momentum"] == 0.5
