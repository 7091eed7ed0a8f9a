"""8-bit integers with a scale for each row (bflow_amd/int8.py, csrc/int8_gemm.hip) and the correlation volume built on them, against 64 bits.

Whole numbers are compared exactly.  The sums of a product are exact, so an element is off by the roundings that follow: sum to 32 bits, alpha * scale_a,
the two products with the scales: 4 * 2^-24, and half a step of the type it is stored in (fp16 2^-11, bf16 2^-8; 32 bits: the last product's own)."""
import math

import numpy as np
import pytest
import torch

import bflow_amd
from bflow_amd import hip, int8
from bflow_amd.corr import CorrBlockParallelMultiTarget, CorrComputation

DEV = "cuda:0"
gpu = pytest.mark.gpu
STEP = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
KINDS = list(STEP)


def quantised(x):
    """(..., K) -> whole numbers and scales by the definition, 64 bits."""
    x = x.double()
    most = x.abs().amax(-1, keepdim=True)
    q = torch.where((most > 0) & torch.isfinite(most), torch.round(127 * x / most), torch.zeros_like(x))
    return q, (most.squeeze(-1).float() / 127)


def rows(r, k, seed=0, batch=()):
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(-128, 128, tuple(batch) + (r, k), generator=g, dtype=torch.int8)
    return q, torch.rand(tuple(batch) + (r,), generator=g) + 0.01


def product(a, sa, b, sb, alpha=1.0):
    return (a.double() @ b.double().transpose(-1, -2)) * sa.double().unsqueeze(-1) * sb.double().unsqueeze(-2) * alpha


def check(got, want, kind):
    assert got.dtype == kind and tuple(got.shape) == tuple(want.shape)
    tiny = 2.0 ** -25 if kind == torch.float16 else 0.0         # half the smallest step of an fp16 below its normal range
    lim = want.abs() * (4 * 2.0 ** -24 + STEP[kind]) + tiny
    bad = (got.cpu().double() - want).abs() > lim
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist())


# ------------------------------------------------------------------------------------------------------------------------- refusals (CPU)
def test_refuses_what_it_cannot_take():
    q, s = rows(4, 16)
    with pytest.raises(hip.BflowHipError, match="no CPU fallback"):
        int8.quantize_rows(torch.zeros(4, 4))
    with pytest.raises(hip.BflowHipError, match="no CPU fallback"):
        int8.quantize_pixels(torch.zeros(16, 4, 4))
    with pytest.raises(hip.BflowHipError, match="no CPU fallback"):
        int8.matmul(q, s, q, s)
    with pytest.raises(hip.BflowHipError, match="same length"):
        int8.matmul(q, s, q[:, :8], s)
    with pytest.raises(hip.BflowHipError, match="scale for each row"):
        int8.matmul(q, s[:3], q, s)
    with pytest.raises(hip.BflowHipError, match="maps"):
        int8.quantize_pixels(torch.zeros(4, 4))


def test_c_entries_refuse_bad_arguments():
    """The C entries' own checks, before any launch: no GPU is touched."""
    lib = hip.lib()
    names = ("a b scale_a scale_b out a_stride0 a_stride1 b_stride0 b_stride1 sa_stride0 sa_stride1 sb_stride0 sb_stride1 out_stride0 out_stride1 ldo "
             "lda ldb M N K batch0 batch1 dtype alpha").split()
    fine = dict(dict.fromkeys(names, 0), a=256, b=256, scale_a=256, scale_b=256, out=256, ldo=8, lda=16, ldb=16, M=4, N=8, K=16, batch0=1, batch1=1, alpha=1.0)
    for kw in (dict(a=0), dict(b=0), dict(scale_a=0), dict(scale_b=0), dict(out=0), dict(M=0), dict(N=-1), dict(K=0), dict(batch0=0), dict(batch1=0), dict(dtype=3), dict(lda=15), dict(ldb=0),
               dict(lda=24), dict(a=264), dict(b=257), dict(a_stride0=8), dict(b_stride1=4), dict(ldo=7), dict(K=131072, lda=131072, ldb=131072), dict(lda=(1 << 22) + 16),
               dict(batch0=256, batch1=256)):
        v = {**fine, **kw}
        assert lib.bflow_i8_gemm(hip.I8_GEMM.pack(*(v[n] for n in names)), None) < 0, kw
        assert b"i8_gemm" in lib.bflow_last_error_string()
    assert lib.bflow_i8_gemm(None, None) < 0
    for item in ((0, 256, 8, 4, 8, 16), (256, 0, 8, 4, 8, 16), (256, 260, 8, 4, 8, 16), (256, 256, 8, 0, 8, 16), (256, 256, 8, 4, 0, 16), (256, 256, 8, 4, 8, 8), (256, 256, 8, 4, 20, 16)):
        assert lib.bflow_i8_pad_rows(hip.I8_PAD.pack(*item), 1, None) == -1, item
    assert lib.bflow_i8_pad_rows(None, 1, None) == -1 and lib.bflow_i8_pad_rows(hip.I8_PAD.pack(256, 256, 8, 4, 8, 16), 3, None) == -1
    for kw in (dict(x=0), dict(q=0), dict(s=0), dict(rows=0), dict(K=0), dict(ldq=8), dict(ldq=24), dict(q=260), dict(dtype=5), dict(ld=-1)):
        v = {**dict(x=256, dtype=0, ld=16, rows=4, K=16, q=256, ldq=16, s=256), **kw}
        assert lib.bflow_i8_quantize_rows(v["x"], v["dtype"], v["ld"], v["rows"], v["K"], v["q"], v["ldq"], v["s"], None) == -1, kw
    for kw in (dict(x=0), dict(hi=256), dict(q=0), dict(s=0), dict(q=264), dict(B=0), dict(D=24), dict(D=0), dict(h=0), dict(x=0, hi=256, lo=256, np=15), dict(x=0, hi=256, lo=256, D=16)):
        v = {**dict(x=256, hi=0, lo=0, np=128, B=1, D=32, h=4, w=4, q=256, s=256), **kw}
        assert lib.bflow_i8_quantize_pixels(v["x"], v["hi"], v["lo"], v["np"], v["B"], v["D"], v["h"], v["w"], 0, v["q"], v["s"], None) == -1, kw


def test_precision_names():
    from bflow_amd import corr
    f1, f2 = torch.zeros(1, 96, 4, 8), torch.zeros(2, 1, 96, 4, 8)
    c = CorrComputation(f1, f2, [1, 1])
    assert c.tiled_supported("i8") and c.tiled_supported("i8/w") and not c.pool1_fusable("i8")
    assert not CorrComputation(torch.zeros(1, 48, 4, 8), torch.zeros(1, 1, 48, 4, 8), [1]).tiled_supported("i8")
    with pytest.raises(hip.BflowHipError, match="tiled"):
        c.get_correlation_volume(tiled=False, precision="i8")
    assert corr.check_precision("i8/w") == "i8/w"


# --------------------------------------------------------------------------------------------------------------------------- quantisation
@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("r,k", [(1, 1), (3, 15), (5, 16), (4, 17), (300, 567), (7, 64), (2, 4099), (9, 1000)])
def test_quantize_rows(r, k, kind):
    x = (torch.randn(r, k, generator=torch.Generator().manual_seed(r + k)) * torch.logspace(-6, 6, r).unsqueeze(1)).to(kind)
    if kind == torch.float16:
        x = x.clamp(-60000, 60000)
    q, s = int8.quantize_rows(x.to(DEV))
    want, scale = quantised(x)
    assert q.dtype == torch.int8 and q.shape == x.shape and (r == 1 or q.stride(0) % 16 == 0)
    assert torch.equal(q.cpu().double(), want) and torch.equal(s.cpu(), scale)
    whole = torch.as_strided(q, (r, (k + 15) // 16 * 16), ((k + 15) // 16 * 16, 1))
    assert not whole[:, k:].any()


@gpu
def test_quantize_halves_and_neighbours():
    """127 x / max next to and on halves: on a half to the even number, beside it to the near one, also where 32 bits cannot tell."""
    halves = torch.arange(-126, 127).float() + 0.5
    up, down = torch.nextafter(halves, torch.full_like(halves, 1e9)), torch.nextafter(halves, torch.full_like(halves, -1e9))
    row = torch.cat([torch.tensor([127.0]), halves, up, down])
    x = torch.stack([row * f for f in (1.0, 2.0 ** -100, 2.0 ** 100, 3.0, 1.0 / 3.0, 1e-35, 1e-38, 1e-44)])
    q, s = int8.quantize_rows(x.to(DEV))
    want, scale = quantised(x)
    assert torch.equal(q.cpu().double(), want) and torch.equal(s.cpu(), scale)
    assert want[0, 1:254].remainder(2).abs().max() == 0
    many = torch.randn(400, 2000, generator=torch.Generator().manual_seed(5))
    q, _ = int8.quantize_rows(many.to(DEV))
    assert torch.equal(q.cpu().double(), quantised(many)[0])


@gpu
def test_quantize_lost_values_and_strides():
    x = torch.randn(6, 40)
    x[0], x[1, 3], x[2, 39], x[3, 0] = 0.0, float("inf"), float("nan"), float("-inf")
    q, s = int8.quantize_rows(x.to(DEV))
    assert not q[:4].any() and s[0] == 0 and s[1] == float("inf") and torch.isnan(s[2]) and s[3] == float("inf")
    assert torch.equal(q[4:].cpu().double(), quantised(x[4:])[0])
    y = int8.matmul(q, s, q, s).cpu()
    assert torch.isnan(y[1:4]).all() and torch.isnan(y[:, 1:4]).all() and not y[0, [0, 4, 5]].any() and torch.isfinite(y[4:, 4:]).all()
    big = torch.randn(3, 50, 70)
    dev = big.to(DEV)
    for d, c in ((dev[:, 3:20, 5:], big[:, 3:20, 5:]), (dev.transpose(1, 2), big.transpose(1, 2)), (dev[1, 2], big[1, 2]), (dev[..., ::2], big[..., ::2]),
                 (dev[:1].expand(4, 50, 70), big[:1].expand(4, 50, 70))):
        q, s = int8.quantize_rows(d)
        want, scale = quantised(c)
        assert torch.equal(q.cpu().double(), want) and torch.equal(s.cpu(), scale)
    q, s = int8.quantize_rows(dev[:, :0])
    assert q.shape == (3, 0, 70) and s.shape == (3, 0)
    q, s = int8.quantize_rows(dev[..., :0])
    assert q.shape == (3, 50, 0) and not s.any()
    with pytest.raises(hip.BflowHipError, match="quantize_rows"):
        int8.quantize_rows(dev.double())


def tile_order(h, w):
    """Pixel of each place of the tiled plane, -1 outside the map."""
    across = -(-w // 8)
    r = torch.arange(hip.tiled_plane_size(h, w))
    y, x = r // 32 // across * 4 + r % 32 // 8, r // 32 % across * 8 + r % 8
    return torch.where((y < h) & (x < w), y * w + x, torch.full_like(r, -1))


@gpu
@pytest.mark.parametrize("B,D,h,w", [(1, 16, 1, 1), (2, 32, 5, 7), (3, 96, 9, 17), (1, 256, 60, 80), (2, 144, 4, 8)])
def test_quantize_pixels(B, D, h, w):
    x = torch.randn(B, D, h, w, generator=torch.Generator().manual_seed(D))
    x[0, :, 0, 0] = 0
    want, scale = quantised(x.flatten(-2).transpose(1, 2))
    q, s = int8.quantize_pixels(x.to(DEV))
    assert torch.equal(q.cpu().double(), want) and torch.equal(s.cpu(), scale)
    order = tile_order(h, w)
    inside = order >= 0
    q, s = int8.quantize_pixels(x.to(DEV), tiled=True)
    assert torch.equal(q.cpu().double()[:, inside], want[:, order[inside]]) and torch.equal(s.cpu()[:, inside], scale[:, order[inside]])
    assert not q[:, ~inside].any() and not s[:, ~inside].any()
    if D % 32 == 0:                                         # the conv engine's operand holds hi + lo * 2^-11: quantised as that value
        p = hip.split_pack(x.flatten(-2).to(DEV))
        held = (p[0].float() + p[1].float() / 2048)[:, :, :h * w].permute(0, 2, 1, 3).reshape(B, h * w, D).cpu()
        want, scale = quantised(held)
        for tiled in (False, True):
            q, s = int8.quantize_packed(p, h, w, tiled)
            at = order[inside] if tiled else slice(None)
            here = inside if tiled else slice(None)
            assert torch.equal(q.cpu().double()[:, here], want[:, at]) and torch.equal(s.cpu()[:, here], scale[:, at])


@gpu
def test_quantize_pixels_refuses():
    with pytest.raises(hip.BflowHipError, match="multiple of 16"):
        int8.quantize_pixels(torch.zeros(24, 4, 4, device=DEV))
    with pytest.raises(hip.BflowHipError):
        int8.quantize_packed(torch.zeros(2, 1, 1, 128, 16, dtype=torch.float16, device=DEV), 4, 4)


# -------------------------------------------------------------------------------------------------------------------------------- product
SIZES = [(1, 1, 1), (1, 5, 16), (3, 2, 15), (1, 4096, 4096), (1, 1000, 777), (2, 130, 300), (16, 64, 128), (17, 63, 127), (64, 64, 129), (65, 70, 256), (200, 3, 1021), (333, 1001, 255),
         (129, 257, 384), (600, 520, 64), (1030, 1100, 200), (5, 9, 20000), (33, 900, 2048)]


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_matmul(m, n, k, kind):
    a, sa = rows(m, k, 1)
    b, sb = rows(n, k, 2)
    if kind == torch.float16:
        sa = sa / (16384 * k) * 100
    y = int8.matmul(a.to(DEV), sa.to(DEV), b.to(DEV), sb.to(DEV), out_dtype=kind, alpha=0.37)
    check(y, product(a, sa, b, sb, float(np.float32(0.37))), kind)


@gpu
def test_matmul_is_exact_at_the_ends():
    """The largest sums that 32 bits hold, and their halves that cancel."""
    k = 131071
    a = torch.full((2, k), -128, dtype=torch.int8)
    a[1, ::2] = 127
    one = torch.ones(2)
    y = int8.matmul(a.to(DEV), one.to(DEV), a.to(DEV), one.to(DEV))
    assert torch.equal(y.cpu().double(), product(a, one, a, one).float().double())
    with pytest.raises(hip.BflowHipError, match="131072"):
        z = torch.zeros(1, k + 1, dtype=torch.int8, device=DEV)
        int8.matmul(z, one[:1].to(DEV), z, one[:1].to(DEV))


@gpu
@pytest.mark.parametrize("ba,bb", [((3,), (3,)), ((3,), ()), ((), (4,)), ((2, 3), (2, 3)), ((3,), (2, 3)), ((2, 1), (2, 3)), ((2, 1, 3), (1, 4, 3)), ((1,), (5,)), ((2, 2, 2, 1), (2,))])
@pytest.mark.parametrize("k", [48, 50])
def test_matmul_broadcasts(ba, bb, k):
    a, sa = rows(37, k, 1, ba)
    b, sb = rows(41, k, 2, bb)
    y = int8.matmul(a.to(DEV), sa.to(DEV), b.to(DEV), sb.to(DEV))
    check(y, product(a, sa, b, sb), torch.float32)


@gpu
def test_matmul_strides_and_out():
    """Rows at any distance, odd starts, transposed and repeated rows; an `out` that is a part of something else: the rest stays as it was."""
    a, sa = rows(90, 200, 1)
    b, sb = rows(80, 200, 2)
    da, dsa, db, dsb = (t.to(DEV) for t in (a, sa, b, sb))
    for s in (np.s_[:, :], np.s_[:, 16:144], np.s_[:, 3:150], np.s_[5:60, 1:], np.s_[::3, :96], np.s_[:, ::2], np.s_[1:2, 7:8]):
        y = int8.matmul(da[s], dsa[s[0]], db[s], dsb[s[0]])
        check(y, product(a[s], sa[s[0]], b[s], sb[s[0]]), torch.float32)
    t, st = rows(200, 64, 3)
    y = int8.matmul(t.to(DEV).t(), torch.ones(64, device=DEV), da, dsa)
    check(y, product(t.t(), torch.ones(64), a, sa), torch.float32)
    y = int8.matmul(da[:1].expand(70, 200), dsa[:1].expand(70), db, dsb)
    check(y, product(a[:1].expand(70, 200), sa[:1].expand(70), b, sb), torch.float32)
    for kind in KINDS:
        room = torch.full((3, 100, 131), 7.0, dtype=kind, device=DEV)
        view = room[1, 4:94, 10:90]
        assert int8.matmul(da, dsa / 4096, db, dsb, out_dtype=kind, out=view) is view
        check(view, product(a, sa / 4096, b, sb), kind)
        view.fill_(7.0)
        assert bool((room == 7.0).all())
    pair = torch.full((4, 2, 96, 80), 7.0, device=DEV)
    int8.matmul(da.view(1, 90, 200).expand(2, 90, 200), dsa.expand(2, 90), db, dsb, out=pair[1:3, 0, 2:92])
    assert bool((pair[:, 1] == 7.0).all()) and bool((pair[1:3, 0, :2] == 7.0).all()) and bool((pair[1:3, 0, 92:] == 7.0).all()) and bool((pair[[0, 3]] == 7.0).all())
    check(pair[2, 0, 2:92], product(a, sa, b, sb), torch.float32)


@gpu
def test_matmul_empty_and_refusals():
    a, sa = (t.to(DEV) for t in rows(5, 32))
    assert int8.matmul(a[:0], sa[:0], a, sa).shape == (0, 5) and int8.matmul(a, sa, a[:0], sa[:0]).shape == (5, 0)
    assert not int8.matmul(a[:, :0], sa, a[:, :0], sa).any()
    for kw, match in ((dict(out_dtype=torch.float64), "out_dtype"), (dict(out=torch.zeros(5, 6, device=DEV)), "out"), (dict(out=torch.zeros(5, 5, device=DEV).t()[:, :]), None),
                      (dict(out=torch.zeros(5, 5)), "out"), (dict(out=torch.zeros(5, 5, device=DEV, dtype=torch.float16)), "out")):
        if match is None:
            with pytest.raises(hip.BflowHipError):
                int8.matmul(a, sa, a, sa, out=torch.zeros(5, 10, device=DEV).t()[:5])
        else:
            with pytest.raises(hip.BflowHipError, match=match):
                int8.matmul(a, sa, a, sa, **kw)
    with pytest.raises(hip.BflowHipError, match="broadcast"):
        int8.matmul(a.expand(2, 5, 32), sa.expand(2, 5), a.expand(3, 5, 32), sa.expand(3, 5))
    with pytest.raises(hip.BflowHipError, match="dtype"):
        int8.matmul(a.float(), sa, a.float(), sa)
    with pytest.raises(hip.BflowHipError, match="dtype"):
        int8.matmul(a, sa.double(), a, sa)


@gpu
def test_matmul_on_streams_and_in_a_graph():
    a, sa = rows(300, 567, 1)
    b, sb = rows(700, 567, 2)
    da, dsa, db, dsb = (t.to(DEV) for t in (a, sa, b, sb))
    x = torch.randn(300, 567, device=DEV)

    def whole():
        q, s = int8.quantize_rows(x)
        return int8.matmul(q, s, db, dsb)
    want, plain = whole(), int8.matmul(da, dsa, db, dsb)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append([whole() for _ in range(3)])
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for ys in got for y in ys)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = whole()
    first = x.clone()
    for k in range(4):
        x.copy_(first if k % 2 else first.flip(0))
        graph.replay()
        assert torch.equal(int8.matmul(da, dsa, db, dsb), plain)
        torch.cuda.synchronize()
        assert torch.equal(out, want if k % 2 else want.flip(0))


# ------------------------------------------------------------------------------------------------------------------------------ the volume
def maps(T, B, D, h, w, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(B, D, h, w, generator=g), torch.randn(T, B, D, h, w, generator=g)


@gpu
@pytest.mark.parametrize("T,B,D,h,w", [(1, 1, 32, 3, 5), (4, 1, 256, 24, 40), (2, 2, 128, 13, 19), (1, 2, 96, 8, 8), (5, 1, 64, 9, 31)])
@pytest.mark.parametrize("name", ["i8", "i8/w"])
def test_volume(T, B, D, h, w, name):
    f1, f2 = maps(T, B, D, h, w)
    vol = CorrComputation(f1.to(DEV), f2.to(DEV), [1] * T).get_correlation_volume(tiled=True, precision=name)
    q1, s1 = quantised(f1.flatten(-2).transpose(-1, -2))
    q2, s2 = quantised(f2.flatten(-2).transpose(-1, -2))
    want = product(q1, s1, q2, s2, float(np.float32(1 / math.sqrt(D))))
    order = tile_order(h, w)
    inside = order >= 0
    assert vol.shape == (T, B, h * w, len(order)) and not vol[..., ~inside].any()
    check(vol[..., inside].contiguous(), want[..., order[inside]], torch.float16 if name == "i8" else torch.float32)


@gpu
def test_block_on_the_8_bit_volume():
    """The whole correlation block (volume, pyramid, look-up) in 8 bits equals the block in fp16 pairs on the maps that the 8 bits stand for."""
    T, B, D, h, w = 2, 1, 128, 16, 24
    f1, f2 = (t.to(DEV) for t in maps(T, B, D, h, w, 3))

    def held(f):
        q, s = int8.quantize_pixels(f)
        return (q.float() * s.unsqueeze(-1)).transpose(-1, -2).reshape(f.shape).contiguous()
    coords = torch.rand(T, B, 2, h, w, device=DEV) * 20 - 2
    a = CorrBlockParallelMultiTarget(CorrComputation(f1, f2, [3, 2]), layout="tiled", precision="i8/w")(coords)
    b = CorrBlockParallelMultiTarget(CorrComputation(held(f1), held(f2), [3, 2]), layout="tiled", precision="split")(coords)
    # sums of 128 products of pairs: 3 * 2^-22 each, against the largest value of the volume
    assert float((a - b).abs().max()) < 3 * 2.0 ** -22 * math.sqrt(D) * float(b.abs().max()) + 1e-6


@gpu
@pytest.mark.parametrize("name", ["i8", "i8/w"])
def test_model_forward_in_8_bits(name):
    """`correlation.precision: i8` through the whole model, eager and as a replayed graph: the packed operands of the encoder are quantised as they are."""
    from bflow_amd import configs, synthetic
    from bflow_amd.weights import deterministic_state_dict
    m = bflow_amd.RAFTSpline(configs.model_config("E_LU4_BD2", {"correlation": {"precision": name}})).eval()
    m.load_state_dict(deterministic_state_dict(m, seed=0))
    m.to(DEV)
    vox = torch.from_numpy(synthetic.voxel_grid(1, 9, 128, 160, seed=7)).to(DEV)
    with torch.inference_mode():
        m.enable_hipgraph(False)
        eager = m(voxel_grid=vox, iters=3, test_mode=True)[1].get_params().clone()
        m.enable_hipgraph()
        for _ in range(3):
            graphed = m(voxel_grid=vox, iters=3, test_mode=True)[1].get_params().clone()
            assert torch.equal(eager, graphed)
    assert bool(torch.isfinite(eager).all())


@gpu
def test_out_that_repeats_itself_is_refused():
    a, sa = (t.to(DEV) for t in rows(5, 32))
    with pytest.raises(hip.BflowHipError, match="out"):
        int8.matmul(a.expand(3, 5, 32), sa.expand(3, 5), a, sa, out=torch.zeros(5, 5, device=DEV).expand(3, 5, 5))


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,n,k", [(4090, 4080, 260), (2201, 2179, 300), (2176, 2178, 128), (1100, 2050, 129), (700, 772, 256), (513, 264, 1), (257, 256, 17), (8192, 33, 70), (40, 5000, 3000)])
def test_matmul_of_every_form(m, n, k, kind):
    """Tiles of each size, whole and odd, the streaming form at its limits (K = 1, 17, 128, 129, 256), against integers on the GPU's 64-bit floats: exact."""
    a, sa = rows(m, k, 3)
    b, sb = rows(n, k, 4)
    sa, sb = sa / (200 * k), sb
    y = int8.matmul(a.to(DEV), sa.to(DEV), b.to(DEV), sb.to(DEV), out_dtype=kind)
    check(y, product(a, sa, b, sb), kind)


@gpu
def test_streaming_form_leaves_the_rest_alone():
    """M, N and K that end inside a chunk, a panel and a segment; an `out` inside a larger buffer, several matrices, a repeated left side."""
    for kind in KINDS:
        a, sa = rows(555, 200, 1)
        b, sb = rows(312, 200, 2, (3,))
        room = torch.full((3, 570, 336), 7.0, dtype=kind, device=DEV)
        view = room[:, 8:563, 8:320]
        int8.matmul(a.to(DEV), (sa / 4096).to(DEV), b.to(DEV), sb.to(DEV), out_dtype=kind, out=view)
        check(view.contiguous(), product(a, sa / 4096, b, sb), kind)
        view.fill_(7.0)
        assert bool((room == 7.0).all())


def test_too_many_places_are_refused():
    """One pixel wide and 2^28 - 1 high: more places than 2^30, in the tiled order.  No GPU is touched."""
    lib = hip.lib()
    assert lib.bflow_i8_quantize_pixels(256, None, None, 0, 1, 16, (1 << 28) - 1, 1, 1, 256, 256, None) < 0
    assert b"places" in lib.bflow_last_error_string()


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("k", [70, 256, 1000])
def test_rows_have_the_same_bits_alone_and_together(k, kind):
    """Every kernel adds whole numbers and applies the scales in one order: a token's row does not depend on the batch it stands in."""
    (a, sa), (b, sb) = rows(600, k, 1), rows(520, k, 2)
    a, sa, b, sb = (t.to(DEV) for t in (a, sa, b, sb))
    whole = int8.matmul(a, sa, b, sb, kind, 0.37)
    for at, n in ((0, 1), (5, 17), (100, 33), (599, 1), (64, 300)):
        assert torch.equal(int8.matmul(a[at:at + n], sa[at:at + n], b, sb, kind, 0.37), whole[at:at + n])
        if at + n <= 520:
            assert torch.equal(int8.matmul(a, sa, b[at:at + n], sb[at:at + n], kind, 0.37), whole[:, at:at + n])


@gpu
def test_quantise_and_multiply_beside_another_stream():
    """Quantisation and products of two streams at once, and twice in one captured graph, as layers behind one another use them."""
    g = torch.Generator().manual_seed(3)
    xs, ws = [torch.randn(n, 200, generator=g).to(DEV) for n in (1, 70, 400)], [torch.randn(200, 200, generator=g).to(DEV) for _ in range(2)]
    qs = [int8.quantize_rows(w) for w in ws]

    def layers(x):
        for q, s in qs:
            x = int8.matmul(*int8.quantize_rows(x), q, s, alpha=1 / 14)
        return x
    want = [layers(x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = []
    for x, st in zip(xs, streams):
        with torch.cuda.stream(st):
            got.append([layers(x) for _ in range(4)])
    torch.cuda.synchronize()
    assert all(torch.equal(y, w) for ys, w in zip(got, want) for y in ys)
    static = [x.clone() for x in xs]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = [layers(x) for x in static]
    for flip in (False, True, False):
        for s, x in zip(static, xs):
            s.copy_(-x if flip else x)
        graph.replay()
        layers(xs[1])
        torch.cuda.synchronize()
        assert all(torch.equal(y, layers(s)) for y, s in zip(out, static))


@gpu
@pytest.mark.parametrize("m,n,k,kind", [(70000, 70008, 64, torch.float16), (70000, 70001, 300, torch.bfloat16), (20, 1 << 27, 16, torch.float16), (1 << 27, 17, 16, torch.float16)],
                         ids=["streamed", "tiles", "few rows", "few columns"])
def test_results_behind_32_bits(m, n, k, kind):
    """Offsets past 2^32 bytes: the corners and the middle of a result of 4 to 10 GB against 64 bits."""
    g = torch.Generator(device=DEV).manual_seed(5)
    a = torch.randint(-128, 128, (m, (k + 15) // 16 * 16), generator=g, device=DEV, dtype=torch.int8)[:, :k]
    b = torch.randint(-128, 128, (n, (k + 15) // 16 * 16), generator=g, device=DEV, dtype=torch.int8)[:, :k]
    sa, sb = torch.rand(m, generator=g, device=DEV) + 0.01, torch.rand(n, generator=g, device=DEV) + 0.01
    y = int8.matmul(a, sa, b, sb, kind, 1e-3)
    for r in (0, m // 2, max(m - 40, 0)):
        for c in (0, n // 2 + 3, max(n - 40, 0)):
            part = [t.cpu() for t in (a[r:r + 40], sa[r:r + 40], b[c:c + 40], sb[c:c + 40])]
            check(y[r:r + 40, c:c + 40], product(*part, 1e-3), kind)
    del y, a, b
    torch.cuda.empty_cache()


@gpu
def test_quantise_behind_32_bits():
    """2^20 + 3 rows of 4100 numbers, 4.3 GB of whole numbers and 8.6 of input."""
    g = torch.Generator(device=DEV).manual_seed(6)
    x = torch.randn((1 << 20) + 3, 4100, generator=g, device=DEV, dtype=torch.float16)
    q, s = int8.quantize_rows(x)
    for r in (0, 1 << 19, (1 << 20) - 5):
        want, scale = quantised(x[r:r + 8].cpu())
        assert torch.equal(q[r:r + 8].cpu().double(), want)
        assert ((s[r:r + 8].cpu().double() - scale.double()).abs() <= scale.double() * 2.0 ** -23).all()
    del x, q, s
    torch.cuda.empty_cache()


def test_maps_entry_refuses_bad_tables():
    """The C entry's own checks, before any launch: no GPU is touched."""
    lib = hip.lib()
    fine = dict(x=256, hi=0, lo=0, q=256, scale=256, np=0, B=2, tiled=0)
    packed = dict(fine, x=0, hi=256, lo=256, np=20)

    def call(*items, count=None, D=32, h=4, w=5):
        return lib.bflow_i8_quantize_maps(b"".join(hip.I8_MAPS.pack(*v.values(), 0) for v in items), len(items) if count is None else count, D, h, w, None)
    assert lib.bflow_i8_quantize_maps(None, 1, 32, 4, 5, None) < 0
    for bad in (call(fine, count=0), call(fine, fine, fine), call(fine, D=17), call(fine, D=0), call(fine, h=0), call(fine, w=-1), call(fine, h=1 << 15, w=1 << 15), call(fine, packed),
                call(dict(fine, x=0)), call(dict(fine, q=0)), call(dict(fine, scale=0)), call(dict(fine, hi=256, lo=256)), call(dict(fine, B=0)), call(dict(fine, B=65536)),
                call(fine, dict(fine, B=65534)), call(dict(packed, np=19)), call(packed, D=48), call(dict(fine, q=264))):
        assert bad < 0 and b"i8_quantize_pixels" in lib.bflow_last_error_string()


@gpu
@pytest.mark.parametrize("B1,B2,D,h,w", [(1, 4, 256, 13, 21), (2, 2, 64, 8, 16), (3, 1, 288, 5, 3), (1, 1, 32, 1, 1)])
def test_both_operands_in_one_launch(B1, B2, D, h, w):
    g = torch.Generator().manual_seed(D + h)
    f1, f2 = torch.randn(B1, D, h, w, generator=g).to(DEV), torch.randn(B2, D, h, w, generator=g).to(DEV)
    f2[0, :, 0, 0] = float("nan")
    want = int8.quantize_pixels(f1) + int8.quantize_pixels(f2, tiled=True)
    got = sum(int8.quantize_operands(f1, f2), ())
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(got, want))
    p1, p2 = (hip.split_pack(f.reshape(f.shape[0], D, h * w).nan_to_num()) for f in (f1, f2))
    want = int8.quantize_packed(p1, h, w) + int8.quantize_packed(p2, h, w, tiled=True)
    got = sum(int8.quantize_operands(p1, p2, (h, w)), ())
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    with pytest.raises(hip.BflowHipError, match="different"):
        int8.quantize_operands(f1, f2[..., :-1] if w > 1 else f2[:, :16])


@gpu
@pytest.mark.parametrize("k,ldd,at,ld", [(17, 32, 0, 17), (17, 32, 1, 19), (16, 32, 3, 16), (1, 16, 2, 1), (3, 48, 1, 5), (567, 576, 0, 567), (30, 32, 3, 31), (48, 48, 1, 48), (13, 64, 0, 40)])
def test_padded_rows_hold_zeros_behind_their_end(k, ldd, at, ld):
    """bflow_i8_pad_rows: the row, then zeros, whatever stands behind it in memory and at whatever address; two operands in a launch, the rest untouched."""
    r = 37
    src = torch.randint(1, 127, (at + r * ld + k,), generator=torch.Generator().manual_seed(k), dtype=torch.int8)
    dev = src.to(DEV)
    room = torch.full((2, r + 2, ldd), 9, dtype=torch.int8, device=DEV)
    lib = hip.lib()
    items = b"".join(hip.I8_PAD.pack(dev.data_ptr() + at, room[i, 1].data_ptr(), ld, r, k, ldd) for i in range(2))
    assert lib.bflow_i8_pad_rows(items, 2, torch.cuda.current_stream().cuda_stream) == 0
    got = room.cpu()
    want = torch.stack([src[at + i * ld:at + i * ld + k] for i in range(r)])
    assert torch.equal(got[0, 1:-1, :k], want) and torch.equal(got[1], got[0])
    assert not got[:, 1:-1, k:].any() and bool((got[:, 0] == 9).all()) and bool((got[:, -1] == 9).all())


def test_sizes_beyond_the_entries_integers_are_refused():
    """Sizes that a C int would cut off, or a kernel's 32-bit loop or a launch cannot count to: an error, before anything is allocated or launched."""
    one, s = torch.zeros(1, 16, dtype=torch.int8), torch.zeros(1)
    for n in ((1 << 31) - 256, (1 << 31) + 5, (1 << 32) + 3):
        for call in (lambda: int8.quantize_rows(torch.zeros(1, 1).expand(1, n)), lambda: int8.matmul(one.expand(n, 16), s.expand(n), one, s),
                     lambda: int8.matmul(one, s, one.expand(n, 16), s.expand(n)), lambda: int8.matmul(one[:, :1].expand(1, n), s, one[:, :1].expand(1, n), s),
                     lambda: int8.quantize_pixels(torch.zeros(1).expand(16, n, 1)), lambda: int8.quantize_pixels(torch.zeros(1).expand(16, 1 << 20, 1 << 12)),
                     lambda: int8.quantize_pixels(torch.zeros(1).expand(n, 1, 1))):
            with pytest.raises(hip.BflowHipError, match="at most"):
                call()
    lib = hip.lib()
    top = (1 << 31) - 1
    for K, ldq in ((top - 15, top - 15), (16, top - 15)):
        assert lib.bflow_i8_quantize_rows(256, 0, K, 4, K, 256, ldq, 256, None) == -2 and b"quantize_rows" in lib.bflow_last_error_string()

    def gemm(M, N):
        return lib.bflow_i8_gemm(hip.I8_GEMM.pack(256, 256, 256, 256, 256, *[0] * 10, N, 16, 16, M, N, 16, 1, 1, 0, 1.0), None)
    for M, N in ((top, 1), (1, top), (top, top), (1 << 28, 3), (32, 1 << 28), (1 << 24, 1 << 24), (top - 511, top - 511)):
        assert gemm(M, N) == -2 and b"i8_gemm" in lib.bflow_last_error_string()
    for h, w, hi in ((1 << 14, (1 << 14) - 1, 0), (1, (1 << 27) + 8, 0), (1, (1 << 28) - 1, 256)):
        assert lib.bflow_i8_quantize_pixels(0 if hi else 256, hi, hi, 1 << 28, 1, 32, h, w, 1, 256, 256, None) == -2 and b"places" in lib.bflow_last_error_string()


@gpu
@pytest.mark.parametrize("T,B,D,h,w", [(1, 1, 32, 3, 5), (4, 1, 256, 24, 40), (2, 3, 128, 13, 19), (3, 2, 256, 9, 31)])
@pytest.mark.parametrize("name", ["i8", "i8/w"])
def test_volume_of_packed_operands(T, B, D, h, w, name):
    """What the model's forward pass builds: the encoder's planes, references and targets of several samples behind one another in one tensor, quantised as the
    values that they hold (hi + lo * 2^-11); against 64 bits, and the block on them against the block on maps of those values."""
    f1, f2 = maps(T, B, D, h, w, 7)
    planes = hip.split_pack(torch.cat([f1, f2.flatten(0, 1)]).flatten(-2).to(DEV))
    held = (planes[0].double() + planes[1].double() / 2048)[:, :, :h * w].permute(0, 2, 1, 3).reshape(B * (1 + T), h * w, D).cpu()
    assert torch.equal(held.float().double(), held)
    (q1, s1), (q2, s2) = quantised(held[:B]), quantised(held[B:].view(T, B, h * w, D))
    want = product(q1, s1, q2, s2, float(np.float32(1 / math.sqrt(D))))
    kind = torch.float16 if name == "i8" else torch.float32
    packed = lambda: CorrComputation.from_packed(planes[:, :B], planes[:, B:], B, D, h, w, [2] * T)
    vol = packed().get_correlation_volume(tiled=True, precision=name)
    order = tile_order(h, w)
    inside = order >= 0
    assert vol.shape == (T, B, h * w, len(order)) and not vol[..., ~inside].any()
    check(vol[..., inside].contiguous(), want[..., order[inside]], kind)
    room = torch.empty_like(vol)
    assert packed().get_correlation_volume(tiled=True, precision=name, out=room) is room and torch.equal(room, vol)
    as_maps = held.float().transpose(1, 2).reshape(-1, D, h, w).to(DEV).contiguous()
    plain = CorrComputation(as_maps[:B], as_maps[B:].view(T, B, D, h, w), [2] * T)
    coords = torch.rand(T, B, 2, h, w, generator=torch.Generator().manual_seed(1)).to(DEV) * max(h, w)
    blocks = [CorrBlockParallelMultiTarget(c, layout="tiled", precision=name)(coords) for c in (packed(), plain)]
    assert torch.equal(*blocks)
