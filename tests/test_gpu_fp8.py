"""Block-scaled 8-bit operands, their products, and the FP8 expert layer, against plain 64-bit forms.

Quantising is exact: the scale is max / 448 rounded once to fp32, the code the nearest of the exact quotient.
Products: codes multiply exactly, a block's 128 products are added in fp32 or a form that drops at most one unit in the
last place per addition, 2^-23 of the magnitudes added; then two scales (two roundings) and one fp32 addition per block.
Every term meets at most 128 + blocks + 3 of these, so a sum is off by at most that many 2^-23 of its terms' magnitudes;
then it is rounded to the output's type, half a step = finfo.eps / 2 (and half the smallest subnormal)."""
import pytest
import torch

from tests import fp8_plain as P
from xcaliber_b200 import fp8, ops, synth

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def half_step(t):
    return torch.finfo(t).eps / 2, torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def assert_near(got, ref, tol):
    d = (got.double() - ref).abs()
    assert bool((d <= tol).all()), f"off by {float((d - tol).max()):.3g} more than allowed"


def assert_quant(codes, scale, x):
    q, s = P.quant(x)
    assert torch.equal(scale.double(), s)
    assert torch.equal(codes.double(), q)


# ---- quantising ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k", [(1, 1), (1, 7168), (3, 127), (2, 129), (5, 2880), (130, 200), (1000, 512), (7, 15), (3000, 130)])
def test_quant_is_exact(m, k, dtype):
    torch.manual_seed(m + k)
    x = (torch.randn(m, k, device="cuda") * torch.randint(1, 40, (1, k), device="cuda")).to(dtype)
    codes, scale = fp8.quant(x)
    assert codes.shape == (m, k) and codes.dtype == torch.float8_e4m3fn and scale.shape == (m, P.blocks(k))
    assert_quant(codes, scale, x)


def test_quant_at_the_borders_of_codes():
    """Every midpoint of two codes and its neighbours in fp32, with scales that are powers of two (quotients exactly on the
    border) and that are not (quotients next to it), down to tiny and up to huge blocks."""
    v = P.e4m3_values()
    mid = ((v[1:] + v[:-1]) / 2).float()
    near = torch.cat([mid, mid.nextafter(torch.tensor(1e9)), mid.nextafter(torch.tensor(0.0)), v.float()])
    near = torch.cat([near, near.new_zeros(-near.numel() % 127)]).view(-1, 127)
    rows = torch.cat([torch.full((near.shape[0], 1), 448.0), near], 1)
    for f in (1.0, 2.0 ** -8, 1.1, 0.3333, 7e-5, 1e-30, 2.0 ** -120, 3e-38, 1e-42, 3e35):
        x = (rows * f).cuda()
        codes, scale = fp8.quant(x)
        assert_quant(codes, scale, x)
        codes, scale = fp8.quant(-x)
        assert_quant(codes, scale, -x)
    half = (rows * 0.25).half().cuda()
    assert_quant(*fp8.quant(half), half)


def test_quant_of_zeros_infinities_and_nan():
    x = torch.randn(4, 512, device="cuda")
    x[0, 128:256] = 0
    x[1, 200], x[2, 300], x[3, 511] = float("inf"), float("nan"), float("-inf")
    codes, scale = fp8.quant(x)
    assert float(scale[0, 1]) == 0 and not codes[0, 128:256].float().any()
    assert float(scale[1, 1]) == float("inf") and bool(scale[2, 2].isnan()) and float(scale[3, 3]) == float("inf")
    bad = torch.zeros(4, 4, dtype=torch.bool, device="cuda")
    bad[1, 1] = bad[2, 2] = bad[3, 3] = True
    assert torch.equal(codes.float().isnan(), bad.repeat_interleave(128, 1))
    fine = torch.where(bad.repeat_interleave(128, 1), 0, x)
    q, s = P.quant(fine)
    assert torch.equal(codes.double().nan_to_num(0.0), q) and torch.equal(torch.where(bad, 0, scale).double(), s)


@pytest.mark.parametrize("n,e,k,h,dropped", [(1, 8, 2, 4096, 0.0), (16, 256, 8, 7168, 0.0), (33, 8, 3, 200, 0.3), (700, 16, 4, 130, 0.1)])
def test_quant_into_sorted_rows(n, e, k, h, dropped):
    row, _, _, r = P.plan(n, e, k, seed=n, dropped=dropped)
    plan = row.cuda()
    wide = torch.randn(n, h + 5, device="cuda").bfloat16()
    x = wide[:, :h]  # rows of another stride, not 16-byte aligned
    whole = fp8.quant(x)
    assert_quant(*whole, x)
    sorted_ = fp8.quant(x, plan, r)
    t, s = torch.nonzero(plan >= 0, as_tuple=True)
    at = plan[t, s].long()
    for got, one in zip(sorted_, whole):
        want = torch.zeros_like(got, dtype=torch.float32)
        want[at] = one.float()[t]
        assert torch.equal(got.float(), want)
    out = fp8.empty_rows(r, h, "cuda")
    out[0].view(torch.uint8).fill_(0x55)
    out[1].fill_(-7.0)
    fp8.quant(x, plan, out=out)
    left = torch.ones(r, dtype=torch.bool, device="cuda")
    left[at] = False
    assert bool((out[0].view(torch.uint8)[left] == 0x55).all()) and bool((out[1][left] == -7.0).all())
    assert torch.equal(out[0].float()[at], sorted_[0].float()[at]) and torch.equal(out[1][at], sorted_[1][at])


def test_empty_calls():
    x = torch.randn(4, 256, device="cuda").bfloat16()
    none = torch.empty(0, 2, dtype=torch.int32, device="cuda")
    for codes, scale in (fp8.quant(x[:0]), fp8.quant(x[:0], none, 0), fp8.glu_quant(torch.cat([x, x], 1)[:0])):
        assert codes.shape == (0, 256) and scale.shape == (0, 2)
    codes, scale = fp8.quant(x[:0], none, 128)
    assert codes.shape == (128, 256) and not codes.float().any() and not scale.any()
    assert fp8.glu_backward(x[:0], torch.cat([x, x], 1)[:0]).shape == (0, 512)
    codes, scale = fp8.quant_weight(torch.empty(0, 128, 256, device="cuda"))
    assert codes.shape == (0, 128, 256) and scale.shape == (0, 1, 2)
    wq = fp8.quant_weight(torch.randn(2, 128, 256, device="cuda"))
    c, o = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    assert fp8.grouped_matmul(*fp8.quant(x[:0]), *wq, c, o).shape == (0, 128)


def test_quant_leaves_the_padding_of_a_row():
    """130 columns lie in rows of 144 bytes: the 14 bytes behind them are not written."""
    x = torch.randn(9, 130, device="cuda")
    room = torch.full((9, 144), 0x33, dtype=torch.uint8, device="cuda")
    out = (room.view(torch.float8_e4m3fn)[:, :130], fp8.empty_rows(9, 130, "cuda")[1])
    fp8.quant(x, out=out)
    assert bool((room[:, 130:] == 0x33).all())
    assert_quant(*out, x)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(128, 128), (1, 1), (300, 200), (2, 129, 130), (3, 64, 4096)])
def test_quant_weight_is_exact(shape, dtype):
    w = (torch.randn(*shape, device="cuda") * 0.02).to(dtype)
    codes, scale = fp8.quant_weight(w)
    assert codes.shape == w.shape and scale.shape == (*shape[:-2], P.blocks(shape[-2]), P.blocks(shape[-1]))
    n, k = shape[-2:]
    for c, s, m in zip(codes.reshape(-1, n, k), scale.reshape(-1, *scale.shape[-2:]), w.reshape(-1, n, k)):
        for i in range(P.blocks(n)):
            for j in range(P.blocks(k)):
                part = m[i * 128:(i + 1) * 128, j * 128:(j + 1) * 128].double()
                ref = (part.abs().max() / 448).float()
                assert s[i, j] == ref
                assert torch.equal(c[i * 128:(i + 1) * 128, j * 128:(j + 1) * 128].double(), P.e4m3_round(part / ref.double()))


# ---- the gated activation --------------------------------------------------------------------------------------------
def _act_error(name, g, alpha):
    """How far, relative to its value, the fp32 activation may be off: expf 2 units (CUDA's bound), 1 + e half of one, the
    reciprocal 1, four products: below 8 units of 2^-23; the exponent's argument z is off by up to 4 units relative (four
    operations), which multiplies the result by 1 + 4 |z| units."""
    z = {"silu": g, "swiglu_clamp": alpha * g.clamp(max=7.0), "gelu_tanh": 1.6 * (g + 0.044715 * g ** 3)}[name]
    return (8 + 4 * z.abs()) * 2.0 ** -23


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", ["silu", "swiglu_clamp", "gelu_tanh"])
@pytest.mark.parametrize("n,e,k,inter", [(1, 8, 2, 512), (40, 8, 2, 200), (300, 16, 4, 2880), (17, 4, 1, 13)])
def test_glu_quant_and_gradient(n, e, k, inter, name, dtype):
    _, counts, offsets, r = P.plan(n, e, k, seed=n)
    c, o = counts.cuda(), offsets.cuda()
    live = torch.zeros(r, dtype=torch.bool)
    for a, b in zip(offsets.tolist(), counts.tolist()):
        live[a:a + b] = True
    live = live.cuda()
    h = (torch.randn(r, 2 * inter, device="cuda") * 3).to(dtype)
    h[~live] = float("nan")  # not read
    da = torch.randn(r, inter, device="cuda").to(dtype)
    out = fp8.empty_rows(r, inter, "cuda")
    out[0].view(torch.uint8).fill_(0x11)
    out[1].fill_(-3.0)
    codes, scale = fp8.glu_quant(h, name, counts=c, offsets=o, out=out)
    assert bool((codes.view(torch.uint8)[~live] == 0x11).all()) and bool((scale[~live] == -3.0).all())
    g, u = h[live].double().split(inter, 1)
    v = P.act(name, g, u)
    err = _act_error(name, g, 1.702) * v.abs()
    pad = lambda x: torch.nn.functional.pad(x, (0, P.blocks(inter) * 128 - inter)).view(x.shape[0], -1, 128)  # noqa: E731
    s = scale[live].double()
    top = pad(v.abs()).amax(-1) / 448
    assert_near(s, top, pad(err).amax(-1) / 448 + 2.0 ** -24 * top)
    sb = s.repeat_interleave(128, 1)[:, :inter]
    # a code is the nearest of the fp32 value / scale: half a step of the value (2^-4 of it, or half of 2^-9 below the
    # normal codes; the scale's and the value's own errors can widen a step by a factor 1 + 2^-10 at most)
    assert_near(codes[live].double() * sb, v, ((v.abs() * 2.0 ** -4).maximum(sb * 2.0 ** -10) * (1 + 2.0 ** -10)) + 2 * err)
    whole, wscale = fp8.glu_quant(h[live], name)  # without segments: every row
    assert torch.equal(whole.view(torch.uint8), codes[live].view(torch.uint8)) and torch.equal(wscale, scale[live])

    keep = torch.randn(r, 2 * inter, device="cuda").to(dtype)
    dh = fp8.glu_backward(da, h, name, counts=c, offsets=o, out=keep.clone())
    assert torch.equal(dh[~live], keep[~live])
    g, u = g.clone().requires_grad_(), u.clone().requires_grad_()
    ref = torch.cat(torch.autograd.grad(P.act(name, g, u), (g, u), da[live].double()), 1)
    eps = 1e-6
    dg = (P.act(name, g + eps, u) - P.act(name, g - eps, u)) * da[live].double() / (2 * eps)
    at_border = ((g.abs() - 7).abs() < 1e-4) | ((u.abs() - 7).abs() < 1e-4)
    assert bool(((dg - ref[:, :inter]).abs() <= 1e-6 * (1 + dg.abs()))[~at_border].all())  # the formula is the slope
    # dg = da u s (1 + z' (1 - s)): 1 - s is off by 2^-24 absolutely, z' at most 4 (1 + g^2) times that
    rel, floor = half_step(dtype)
    gd, ud = g.detach(), u.detach()
    size = da[live].double().abs().repeat(1, 2) * torch.cat([(ud.abs() + 1) * (1 + 4 * gd.abs() * (1 + gd * gd)), gd.abs()], 1)
    err = _act_error(name, gd, 1.702).repeat(1, 2) + 4 * 2.0 ** -23
    assert_near(dh[live], ref, rel * ref.abs() + floor + err * size)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("name", ["silu", "swiglu_clamp", "gelu_tanh"])
def test_glu_gradient_of_huge_gates(name, dtype):
    """Gates up to the type's largest: the sigmoid is 0 or 1 there (below e^-100 or above 1 - e^-100), its slope 0, and the
    gradients are da u or 0 and da g or 0, one rounding each of the two products and one to the type."""
    most = torch.finfo(dtype).max
    g = torch.tensor([1e3, 1e6, 3e12, 1.5e13, 1e15, 1e19, 1e25, 1e38, most], device="cuda")
    g = torch.cat([g, -g]).to(dtype)
    i = g.numel()
    u, da = torch.full((i,), 1.5, device="cuda", dtype=dtype), torch.full((i,), 0.125, device="cuda", dtype=dtype)
    dh = fp8.glu_backward(da[None], torch.cat([g, u])[None], name)[0].double()
    up = (g > 0).double()
    want_g = 0.125 * 1.5 * up
    want_u = 0.125 * g.double() * up
    if name == "swiglu_clamp":  # gates above the limit have no gradient and count as the limit, where the sigmoid is not yet 1
        want_g, want_u = 0 * up, 0.125 * 7 * torch.sigmoid(torch.tensor(1.702 * 7.0, dtype=torch.float64)) * up
    rel = half_step(dtype)[0] + (2 + 8 + 4 * 12) * 2.0 ** -23 * (name == "swiglu_clamp") + 2.0 ** -23
    assert_near(dh[:i], want_g, rel * want_g.abs())
    assert_near(dh[i:], want_u, rel * want_u.abs())
    nan = torch.cat([torch.full((8,), float("nan"), device="cuda", dtype=dtype), torch.ones(8, device="cuda", dtype=dtype)])[None]
    dn = fp8.glu_backward(torch.ones(1, 8, device="cuda", dtype=dtype), nan, name)
    assert bool(dn[0, 8:].isnan().all()) and (name == "swiglu_clamp" or bool(dn[0, :8].isnan().all()))


def test_glu_keeps_nan_and_saturates():
    h = torch.zeros(1, 256, device="cuda")
    h[0, 5], h[0, 133] = float("nan"), 1.0
    codes, scale = fp8.glu_quant(h)
    assert bool(scale.isnan().all()) and bool(codes.float().isnan().all())
    h = torch.full((2, 256), 3e4, device="cuda").half()
    h[1, :128] = -200.0  # sigmoid underflows: zeros
    codes, scale = fp8.glu_quant(h)
    assert float((fp8.dequant(codes, scale)[0] / float(h[0, 0]) ** 2 - 1).abs().max()) < 2.0 ** -22  # beyond fp16's range
    assert float(scale[1, 0]) == 0.0


# ---- products --------------------------------------------------------------------------------------------------------
def _operands(m, n, k, e=None, seed=0, transpose=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(m, n if transpose else k, generator=g, device="cuda")
    w = torch.randn(*((e,) if e else ()), n, k, generator=g, device="cuda") * 0.02
    return fp8.quant(x), fp8.quant_weight(w)


def _reference(xq, wq, transpose):
    a, w = P.rows64(*xq), P.weight64(*wq)
    w = w if transpose else w.transpose(-1, -2)
    terms = 128 + P.blocks(a.shape[1]) + 3
    return a @ w, terms * 2.0 ** -23 * (a.abs() @ w.abs())


SIZES = [(1, 128, 128), (1, 4096, 7168), (2, 1, 1), (3, 130, 100), (16, 512, 1024), (17, 257, 129), (33, 128, 16), (64, 300, 640),
         (65, 4096, 384), (100, 512, 2880), (129, 1000, 1000), (200, 96, 2048), (257, 384, 4097), (300, 17, 33), (1000, 768, 640),
         (2500, 256, 256)]


@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_matmul(m, n, k, transpose, out):
    xq, wq = _operands(m, n, k, seed=m + n + k, transpose=transpose)
    y = fp8.matmul(*xq, *wq, transpose=transpose, out_dtype=out)
    assert fp8.status() == 0
    ref, err = _reference(xq, wq, transpose)
    rel, floor = half_step(out)
    assert y.dtype == out and y.shape == ref.shape
    assert_near(y, ref, rel * ref.abs() + floor + err)
    assert torch.equal(y, fp8.matmul(*xq, *wq, transpose=transpose, out_dtype=out))  # the same bits on every run


def test_matmul_gradient_is_the_adjoint_and_the_slope():
    """<dy, matmul(x)> = <matmul(dy, transpose), x> for operands that are codes, and both are the slope of the product
    along x (it is linear: the difference of two products is the product of the difference)."""
    m, n, k = 70, 300, 500
    xq, wq = _operands(m, n, k, seed=1)
    dq, _ = _operands(m, n, k, seed=2, transpose=True)
    y = fp8.matmul(*xq, *wq, out_dtype=torch.float32)
    dx = fp8.matmul(*dq, *wq, transpose=True, out_dtype=torch.float32)
    x, d = P.rows64(*xq), P.rows64(*dq)
    both = float((y.double() * d).sum()), float((dx.double() * x).sum())
    size = float(((x.abs() @ P.weight64(*wq).abs().t()) * d.abs()).sum())
    assert abs(both[0] - both[1]) <= 2 * (128 + 4 + 3) * 2.0 ** -23 * size
    vq, _ = _operands(m, n, k, seed=3)
    v = P.rows64(*vq)
    up, down = (P.rows64(*xq) + s * v for s in (1, -1))
    w = P.weight64(*wq)
    slope = float((((up @ w.t()) - (down @ w.t())) / 2 * d).sum())
    assert abs(slope - float((dx.double() * v).sum())) <= (128 + 4 + 3) * 2.0 ** -23 * float(((v.abs() @ w.abs().t()) * d.abs()).sum())


def test_matmul_of_other_strides_scale_layouts_and_poisoned_padding():
    m, n, k = 50, 200, 300
    xq, wq = _operands(m, n, k, seed=4)
    ref = fp8.matmul(*xq, *wq)
    wide = torch.full((m, 512), 0x7f, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)  # NaN behind the rows
    wide.view(torch.uint8)[:, 16:16 + k] = xq[0].view(torch.uint8)
    assert torch.equal(fp8.matmul(wide[:, 16:16 + k], xq[1], *wq), ref)
    wwide = torch.full((n + 3, 336), 0x7f, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    wwide.view(torch.uint8)[1:n + 1, :k] = wq[0].view(torch.uint8)
    assert torch.equal(fp8.matmul(*xq, wwide[1:n + 1, :k], wq[1]), ref)
    assert torch.equal(fp8.matmul(xq[0], xq[1].contiguous(), *wq), ref)            # row-major scales
    assert torch.equal(fp8.matmul(xq[0], xq[1].t().contiguous().t(), *wq), ref)    # 50 rows: not a multiple of 4
    one = fp8.quant(torch.randn(6, 100, device="cuda"))
    w1 = fp8.quant_weight(torch.randn(40, 100, device="cuda"))
    assert torch.equal(fp8.matmul(*one, *w1), fp8.matmul(one[0], one[1].clone(), *w1))
    assert fp8.matmul(xq[0][:0], xq[1][:0], *wq).shape == (0, n)
    out = torch.full((m, n), 5.0, device="cuda", dtype=torch.float16)
    assert fp8.matmul(*xq, *wq, out=out) is out
    assert_near(out, _reference(xq, wq, False)[0], 2.0 ** -10 * out.double().abs() + 1e-4)
    poisoned = (xq[0], xq[1].clone())
    nan_row = torch.zeros(m, k, device="cuda")
    nan_row[7, 0] = float("nan")
    nq = fp8.quant(nan_row)
    y = fp8.matmul(*nq, *wq)
    assert bool(y[7].isnan().all()) and not y[[i for i in range(m) if i != 7]].any()
    assert torch.equal(fp8.matmul(*poisoned, *wq), ref)
    assert fp8.status() == 0


@pytest.mark.parametrize("what", ["scale shape", "width", "weight scale", "out shape", "type", "alignment", "device type"])
def test_matmul_refuses(what):
    (x, s), (w, ws) = _operands(8, 64, 256)
    out = None
    if what == "scale shape":
        s = s[:, :1]
    elif what == "width":
        x = x[:, :128]
    elif what == "weight scale":
        ws = ws[:, :1]
    elif what == "out shape":
        out = torch.empty(8, 65, device="cuda")
    elif what == "type":
        x = x.float()
    elif what == "alignment":
        x = torch.zeros(8, 260, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)[:, 1:257]
    else:
        s = s.cpu()
    with pytest.raises(RuntimeError):
        fp8.matmul(x, s, w, ws, out=out)


def _segments(counts):
    offsets, at = [], 0
    for c in counts:
        offsets.append(at)
        at += -(-c // 128) * 128
    return torch.tensor(counts, dtype=torch.int32, device="cuda"), torch.tensor(offsets + [at], dtype=torch.int32, device="cuda"), max(at, 128)


GROUPS = [([5, 0, 16, 17, 1], 256, 384), ([0, 0, 3], 130, 100), ([128, 129, 300, 0, 64], 300, 640), ([700, 1, 0, 256, 257], 129, 1040),
          ([0] * 60 + [2, 1, 0, 3], 1536, 256), ([33], 512, 128), ([0, 0, 0], 128, 128)]


@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("counts,n,k", GROUPS)
def test_grouped_matmul(counts, n, k, transpose, out):
    c, o, r = _segments(counts)
    (codes, scale), wq = _operands(r, n, k, e=len(counts), seed=n, transpose=transpose)
    live = torch.zeros(r, dtype=torch.bool, device="cuda")
    for a, b in zip(o.tolist(), counts):
        live[a:a + b] = True
    codes.view(torch.uint8)[~live] = 0x7f  # NaN in rows of no expert: read into tiles, stored nowhere
    scale[~live] = float("nan")
    features = k if transpose else n
    rel, floor = half_step(out)
    results = []
    for hint in (0, sum(counts), 1, 100000):
        keep = torch.full((r, features), -7.0, device="cuda", dtype=out)
        y = fp8.grouped_matmul(codes, scale, *wq, c, o, transpose=transpose, rows_in_use=hint, out=keep)
        assert fp8.status() == 0 and bool((y[~live] == -7.0).all())
        results.append(y)
        for e, b in enumerate(counts):
            if b:
                a = int(o[e])
                ref, err = _reference((codes[a:a + b], scale[a:a + b]), (wq[0][e], wq[1][e]), transpose)
                assert_near(y[a:a + b], ref, rel * ref.abs() + floor + err)
    assert not fp8.grouped_matmul(codes, scale, *wq, c, o, transpose=transpose, out_dtype=out)[~live].any()


def test_grouped_matmul_keeps_to_its_buffers():
    """Segments that lie outside the rows, or not at a multiple of 16, count as empty and are reported; one that runs past
    the end is cut there."""
    (codes, scale), wq = _operands(256, 128, 128, e=4)
    counts = torch.tensor([10, 10, 400, 10], dtype=torch.int32, device="cuda")
    offsets = torch.tensor([0, 24, 128, 4096, 0], dtype=torch.int32, device="cuda")
    y = fp8.grouped_matmul(codes, scale, *wq, counts, offsets, out=torch.full((256, 128), -7.0, device="cuda"))
    assert fp8.status() == 0x700 and fp8.status() == 0
    assert bool((y[10:128] == -7.0).all())
    for a, b, e in ((0, 10, 0), (128, 256, 2)):
        ref, err = _reference((codes[a:b], scale[a:b]), (wq[0][e], wq[1][e]), False)
        assert_near(y[a:b], ref, 2.0 ** -24 * ref.abs() + err)
    neg = torch.tensor([-5, 10, 0, 0], dtype=torch.int32, device="cuda")
    at = torch.tensor([0, 0, -16, 0, 0], dtype=torch.int32, device="cuda")
    y = fp8.grouped_matmul(codes, scale, *wq, neg, at, out=torch.full((256, 128), -7.0, device="cuda"))
    assert fp8.status() == 0 and bool((y[10:] == -7.0).all()) and not bool((y[:10] == -7.0).all())


def test_glu_keeps_to_its_buffers():
    """As the products: segments outside the rows are empty, one past the end is cut, negative counts are none."""
    h = torch.randn(64, 256, device="cuda").bfloat16()
    whole = fp8.glu_quant(h)
    counts = torch.tensor([10, 5, 2 ** 30, -7, 2 ** 31 - 1, 3], dtype=torch.int32, device="cuda")
    offsets = torch.tensor([0, -16, 48, 16, 4096, 2 ** 31 - 8, 0], dtype=torch.int32, device="cuda")
    out = fp8.empty_rows(64, 128, "cuda")
    out[0].view(torch.uint8).fill_(0x21)
    out[1].fill_(-1.0)
    fp8.glu_quant(h, counts=counts, offsets=offsets, out=out)
    live = torch.zeros(64, dtype=torch.bool, device="cuda")
    live[:10] = live[48:] = True
    assert torch.equal(out[0].view(torch.uint8)[live], whole[0].view(torch.uint8)[live]) and torch.equal(out[1][live], whole[1][live])
    assert bool((out[0].view(torch.uint8)[~live] == 0x21).all()) and bool((out[1][~live] == -1.0).all())
    da = torch.randn(64, 128, device="cuda").bfloat16()
    dh = fp8.glu_backward(da, h, counts=counts, offsets=offsets, out=torch.full_like(h, 3.0))
    assert torch.equal(dh[live], fp8.glu_backward(da, h)[live]) and bool((dh[~live] == 3.0).all())


def test_overlapping_segments_beyond_what_can_be_counted():
    """1024 experts that all claim the same 2^19 rows: more tiles than 31 bits hold. Reported, nothing is written."""
    r, e, n = 2 ** 19, 1024, 8192
    codes = torch.zeros(r, 16, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    scale = torch.zeros(1, r, device="cuda").t()
    w = torch.zeros(n, 16, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)[None].expand(e, n, 16)
    counts = torch.full((e,), r, dtype=torch.int32, device="cuda")
    offsets = torch.zeros(e + 1, dtype=torch.int32, device="cuda")
    out = torch.full((r, n), 7.0, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(RuntimeError):  # matrices that lie on top of one another are refused
        fp8.grouped_matmul(codes, scale, w, torch.ones(e, n // 128, 1, device="cuda"), counts, offsets, rows_in_use=16, out=out)
    fp8.grouped_matmul(codes, scale, w.contiguous(), torch.ones(e, n // 128, 1, device="cuda"), counts, offsets, rows_in_use=16, out=out)
    assert fp8.status() == 0x700 and bool((out == 7.0).all())


@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("k", [512, 4096])
def test_overlapping_segments_of_few_tiles(k, transpose):
    """Eight experts that all claim the same 64 rows make 32 tiles, more than the 12 that segments without overlap could:
    too few for every SM, so the launch lets clusters share a tile's contraction. Every tile is computed all the same;
    with one matrix in all eight places every row's product is known."""
    m, n, e = 64, 128, 8
    xq, (w, ws) = _operands(m, *((k, n) if transpose else (n, k)), seed=k, transpose=transpose)
    wq = (torch.empty(e, *w.shape, dtype=w.dtype, device="cuda"), ws.expand(e, *ws.shape).contiguous())
    wq[0].view(torch.uint8).copy_(w.view(torch.uint8).expand(e, *w.shape))
    counts = torch.full((e,), m, dtype=torch.int32, device="cuda")
    offsets = torch.zeros(e + 1, dtype=torch.int32, device="cuda")
    out = torch.full((m, n), -7.0, device="cuda")
    y = fp8.grouped_matmul(*xq, *wq, counts, offsets, transpose=transpose, out=out)
    assert fp8.status() == 0
    ref, err = _reference(xq, (w, ws), transpose)
    assert_near(y, ref, 2.0 ** -24 * ref.abs() + err)


def test_rows_far_behind_in_a_large_buffer():
    """Offsets beyond 2^31 elements, in codes, outputs and sorted rows."""
    k, r = 8192, 2 ** 18 + 256
    codes = torch.zeros(r, k, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    scale = torch.zeros(k // 128, r, device="cuda").t()
    x = torch.randn(20, k, device="cuda", dtype=torch.bfloat16)
    plan = (2 ** 18 + torch.arange(20, dtype=torch.int32, device="cuda"))[:, None]
    fp8.quant(x, plan, out=(codes, scale))
    assert_quant(codes[2 ** 18:2 ** 18 + 20], scale[2 ** 18:2 ** 18 + 20], x)
    wq = fp8.quant_weight(torch.randn(1, 8192, k, device="cuda", dtype=torch.bfloat16) * 0.02)
    counts = torch.tensor([20], dtype=torch.int32, device="cuda")
    offsets = torch.tensor([2 ** 18, 2 ** 18 + 128], dtype=torch.int32, device="cuda")
    y = fp8.grouped_matmul(codes, scale, *wq, counts, offsets, rows_in_use=20)
    assert fp8.status() == 0
    ref, err = _reference((codes[2 ** 18:2 ** 18 + 20], scale[2 ** 18:2 ** 18 + 20]), (wq[0][0], wq[1][0]), False)
    assert_near(y[2 ** 18:2 ** 18 + 20], ref, 2.0 ** -8 * ref.abs() + err)
    back = ops.unpermute(y, plan)
    assert torch.equal(back, y[2 ** 18:2 ** 18 + 20])
    rows = ops.permute(back, plan, out=torch.zeros_like(y))
    assert torch.equal(rows, y)


def _registered_calls():
    row, counts, offsets, r = P.plan(12, 4, 2, seed=1)
    plan, c, o, dev, h = row.cuda(), counts.cuda(), offsets.cuda(), "cuda", 256
    x, rows, w = torch.randn(12, h, device=dev), torch.randn(r, h, device=dev), torch.rand(12, 2, device=dev)
    xq, wm = fp8.quant(x, plan, r), torch.randn(4, 128, h, device=dev)
    wq = fp8.quant_weight(wm)
    z = lambda *d: torch.zeros(*d, device=dev)  # noqa: E731
    codes = lambda *d: torch.zeros(*d, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)  # noqa: E731
    return {"permute": (x, plan, z(r, h)), "unpermute": (rows, plan, w, z(12, h)), "unpermute_new": (rows, plan, w),
            "unpermute_backward": (x, rows, plan, w, z(r, h), z(12, 2)),
            "glu_backward": (rows[:, :128].contiguous(), rows, 0, 1.702, 7.0, c, o, z(r, h)),
            "fp8_quant": (x, plan, codes(r, h), fp8.empty_rows(r, h, dev)[1].zero_()),
            "fp8_quant_weight": (wm, codes(4, 128, h), z(4, 1, 2)),
            "glu_fp8_quant": (rows, 0, 1.702, 7.0, c, o, codes(r, h // 2), fp8.empty_rows(r, h // 2, dev)[1].zero_()),
            "fp8_matmul": (*xq, wq[0][0], wq[1][0], False, z(r, 128)),
            "fp8_matmul_new": (*xq, wq[0][0], wq[1][0], False, torch.bfloat16),
            "fp8_grouped_matmul": (*xq, *wq, c, o, False, 0, z(r, 128))}


@pytest.mark.parametrize("name", ["permute", "unpermute", "unpermute_new", "unpermute_backward", "glu_backward", "fp8_quant",
                                  "fp8_quant_weight", "glu_fp8_quant", "fp8_matmul", "fp8_matmul_new", "fp8_grouped_matmul"])
def test_registered_ops_hold_to_their_schemas(name):
    """What torch asks of a registered op: it changes what its schema says and nothing else, its fake form has the real
    one's results, and it traces. (The schema check multiplies its inputs, which torch cannot do for 8-bit floats.)"""
    args = _registered_calls()[name]
    op = getattr(torch.ops.xmoe_b200, name).default
    tests = ["test_autograd_registration", "test_faketensor", "test_aot_dispatch_dynamic"]
    if not any(isinstance(a, torch.Tensor) and a.dtype == torch.float8_e4m3fn for a in args):
        tests.append("test_schema")
    torch.library.opcheck(op, args, test_utils=tests)


def test_autograd_sees_writes_into_out():
    from tests.test_fp8_cpu import assert_writes_are_seen

    assert_writes_are_seen("cuda")
    with torch.inference_mode():  # buffers that autograd does not track can be written anywhere
        x, out = torch.ones(4, 64, device="cuda"), fp8.empty_rows(4, 64, "cuda")
    fp8.quant(x, out=out)
    assert_quant(*out, x)


# ---- together: the layer ---------------------------------------------------------------------------------------------
SHAPES = {
    "flat": synth.MoEShape("fp8_flat", 512, 384, 8, 2),
    "odd": synth.MoEShape("fp8_odd", 320, 224, 16, 4, activation="swiglu_clamp"),
    "shared": synth.MoEShape("fp8_shared", 256, 256, 32, 4, scoring="sigmoid", num_shared_experts=1, n_group=4, topk_group=2,
                             routed_scale=2.5, router_bias=True),
}


def _layer(shape, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w13 = torch.randn(shape.e_tot, 2 * shape.inter, shape.hidden, generator=g, device="cuda") * shape.hidden ** -0.5
    w2 = torch.randn(shape.e_tot, shape.hidden, shape.inter, generator=g, device="cuda") * shape.inter ** -0.5
    bias = torch.randn(shape.num_experts, generator=g, device="cuda") * 0.01 if shape.router_bias else None
    return fp8.Fp8MoE.from_weights(shape, w13, w2, bias)


def _layer_plain(layer, x, idx, w, dy=None):
    """Token by expert in 64 bits, rounding where the layer rounds: h and the experts' rows to bf16, activations to codes."""
    sh = layer.shape
    n, shared = x.shape[0], sh.num_shared_experts
    idx = torch.cat([idx.long(), torch.arange(sh.num_experts, sh.e_tot, device="cuda").expand(n, -1)], 1)
    w = torch.cat([w.double(), torch.ones(n, shared, dtype=torch.float64, device="cuda")], 1)
    w13, w2 = P.weight64(layer.w13, layer.w13_scale), P.weight64(layer.w2, layer.w2_scale)
    a = P.rows64(*P.quant(x))
    y = torch.zeros(n, sh.hidden, dtype=torch.float64, device="cuda")
    dx, dw = torch.zeros_like(y), torch.zeros_like(w)
    for e in range(sh.e_tot):
        t, s = torch.nonzero(idx == e, as_tuple=True)
        if not len(t):
            continue
        h = (a[t] @ w13[e].t()).bfloat16().double()
        g, u = h.split(sh.inter, 1)
        v = P.act(sh.activation, g, u, sh.swiglu_alpha, sh.swiglu_limit)
        rows = (P.rows64(*P.quant(v.float())) @ w2[e].t()).bfloat16().double()
        y.index_add_(0, t, rows * w[t, s][:, None])
        if dy is not None:
            dw[t, s] = (rows * dy.double()[t]).sum(1)
            drows = (dy.double()[t] * w[t, s][:, None]).bfloat16()
            da = (P.rows64(*P.quant(drows)) @ w2[e]).bfloat16().double()
            gl, ul = g.clone().requires_grad_(), u.clone().requires_grad_()
            dh = torch.cat(torch.autograd.grad(P.act(sh.activation, gl, ul, sh.swiglu_alpha, sh.swiglu_limit), (gl, ul), da), 1)
            dx.index_add_(0, t, (P.rows64(*P.quant(dh.bfloat16())) @ w13[e]).bfloat16().double())
    return (y, dx, dw[:, :sh.top_k]) if dy is not None else y


def _far(a, b):
    return float((a.detach().double() - b).norm() / b.norm())


# The reference rounds where the layer rounds, so what is left is the rounding of the result (at most half a step, 2^-8 of
# every value) and values that lie so near a border of two bf16 numbers that fp32 and 64 bits fall on different sides: their
# share is the ratio of the two errors, about 2^-20 * 16 / 2^-8, and each moves by 2^-7: below 2^-10 of the whole.
FORWARD, BACKWARD = 2.0 ** -8 + 2.0 ** -10, 2.0 ** -8 + 2.0 ** -9


@pytest.mark.parametrize("name", list(SHAPES))
@pytest.mark.parametrize("n", [1, 16, 300])
def test_layer_forward_and_gradients(name, n):
    shape = SHAPES[name]
    layer = _layer(shape)
    torch.manual_seed(n)
    x = torch.randn(n, shape.hidden, device="cuda").bfloat16()
    logits = torch.randn(n, shape.num_experts, device="cuda").bfloat16()
    y = layer.forward(x, logits)
    idx, w = ops.router_topk(logits, shape, layer)
    assert _far(y, _layer_plain(layer, x, idx, w)) <= FORWARD
    dropped = idx.clone()
    if n > 1:
        dropped[::3, 0] = -1
    xg, wg = x.clone().requires_grad_(), w.float().requires_grad_()
    dy = torch.randn(n, shape.hidden, device="cuda").bfloat16()
    y = layer.forward_routed(xg, dropped, wg)
    gx, gw = torch.autograd.grad(y, (xg, wg), dy)
    ry, rx, rw = _layer_plain(layer, x, dropped, w.float(), dy)
    assert _far(y, ry) <= FORWARD and _far(gx, rx) <= BACKWARD and _far(gw, rw) <= BACKWARD
    assert not gw[dropped < 0].any()
    assert fp8.status() == 0


def test_layer_with_an_expert_twice_and_with_nothing():
    """A token may name an expert twice (two slots, two rows, weights add up); a batch may have no slot left at all."""
    shape = SHAPES["flat"]
    layer = _layer(shape)
    torch.manual_seed(9)
    n = 37
    x = torch.randn(n, shape.hidden, device="cuda").bfloat16().requires_grad_()
    w = torch.rand(n, 2, device="cuda").requires_grad_()
    dy = torch.randn(n, shape.hidden, device="cuda").bfloat16()
    twice = torch.randint(0, shape.num_experts, (n, 1), device="cuda", dtype=torch.int32).expand(n, 2).contiguous()
    y = layer.forward_routed(x, twice, w)
    gx, gw = torch.autograd.grad(y, (x, w), dy)
    ry, rx, rw = _layer_plain(layer, x.detach(), twice, w.detach(), dy)
    assert _far(y, ry) <= FORWARD and _far(gx, rx) <= BACKWARD and _far(gw, rw) <= BACKWARD
    none = torch.full((n, 2), -1, dtype=torch.int32, device="cuda")
    y = layer.forward_routed(x, none, w)
    gx, gw = torch.autograd.grad(y, (x, w), dy)
    assert not y.any() and not gx.any() and not gw.any() and fp8.status() == 0


@pytest.mark.parametrize("name", list(SHAPES))
def test_layer_without_tokens_stays_in_the_graph(name):
    """A rank whose share of a batch is empty takes its backward step like the others."""
    shape = SHAPES[name]
    layer = _layer(shape)
    x = torch.empty(0, shape.hidden, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    w = torch.empty(0, shape.top_k, device="cuda", requires_grad=True)
    idx = torch.empty(0, shape.top_k, dtype=torch.int32, device="cuda")
    y = layer.forward_routed(x, idx, w)
    assert y.shape == (0, shape.hidden) and y.dtype == torch.bfloat16
    gx, gw = torch.autograd.grad(y.sum(), (x, w))
    assert gx.shape == x.shape and gw.shape == w.shape and gw.dtype == w.dtype
    y = layer.forward(x, torch.empty(0, shape.num_experts, device="cuda", dtype=torch.bfloat16))
    assert torch.autograd.grad(y.sum(), x)[0].shape == x.shape and fp8.status() == 0


def test_products_in_flight_together():
    """Large and small products (CTA pairs, clusters that share a tile, plain CTAs) on three streams at once."""
    jobs = [_operands(700, 2048, 1024, seed=1), _operands(3, 512, 4096, seed=2), _operands(40, 3000, 512, seed=3)]
    want = [fp8.matmul(*x, *w) for x, w in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    got = [[] for _ in jobs]
    for _ in range(20):
        for (x, w), s, g in zip(jobs, streams, got):
            with torch.cuda.stream(s):
                g.append(fp8.matmul(*x, *w))
    torch.cuda.synchronize()
    for g, ref in zip(got, want):
        assert all(torch.equal(y, ref) for y in g)
    assert fp8.status() == 0


def test_layer_on_another_stream_and_in_two_graphs():
    """Two captured graphs of the same layer and an eager call, in flight together, do not disturb one another."""
    shape = SHAPES["flat"]
    layer = _layer(shape)
    g = torch.Generator(device="cuda").manual_seed(3)
    xs = [torch.randn(64, shape.hidden, generator=g, device="cuda").bfloat16() for _ in range(3)]
    ls = [torch.randn(64, shape.num_experts, generator=g, device="cuda").bfloat16() for _ in range(3)]
    want = [layer.forward(x, lo) for x, lo in zip(xs, ls)]
    graphs, outs = [], []
    for x, lo in zip(xs[:2], ls[:2]):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            layer.forward(x, lo)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(layer.forward(x, lo))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(5):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        with torch.cuda.stream(streams[2]):
            third = layer.forward(xs[2], ls[2])
        torch.cuda.synchronize()
        for got, ref in zip([*outs, third], want):
            assert torch.equal(got, ref)
    assert fp8.status() == 0


def test_layer_gradients_in_a_captured_graph():
    """The layer's forward and backward captured once and replayed on other inputs and routes give the eager calls' bits."""
    shape = SHAPES["odd"]
    layer = _layer(shape)
    n = 50

    def step(x, idx, w, dy):
        y = layer.forward_routed(x, idx, w)
        return (y.detach(), *torch.autograd.grad(y, (x, w), dy))

    def inputs(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        idx = torch.rand(n, shape.num_experts, generator=g, device="cuda").topk(shape.top_k, 1).indices.int()
        return (torch.randn(n, shape.hidden, generator=g, device="cuda").bfloat16(), idx,
                torch.rand(n, shape.top_k, generator=g, device="cuda"),
                torch.randn(n, shape.hidden, generator=g, device="cuda").bfloat16())

    def leaves(i):
        return i[0].requires_grad_(), i[1], i[2].requires_grad_(), i[3]

    fixed = leaves(inputs(0))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(*fixed)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*fixed)
    for seed in (1, 2, 3):
        new = inputs(seed)
        with torch.no_grad():
            for a, b in zip(fixed, new):
                a.copy_(b)
        graph.replay()
        for a, b in zip(got, step(*leaves(new))):
            assert torch.equal(a, b)
    assert fp8.status() == 0


def test_layer_takes_ids_outside_the_experts_as_none():
    shape = SHAPES["flat"]
    layer = _layer(shape)
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(40, shape.hidden, generator=g, device="cuda").bfloat16()
    idx = torch.rand(40, shape.num_experts, generator=g, device="cuda").topk(2, 1).indices.int()
    w = torch.rand(40, 2, generator=g, device="cuda")
    none, outside = idx.clone(), idx.clone()
    none[::3, 1] = -1
    outside[::3, 1] = torch.tensor([8, 9, 1000, -2, -2 ** 31, 2 ** 31 - 1, 8], device="cuda", dtype=torch.int32).repeat(2)
    assert torch.equal(layer.forward_routed(x, outside, w), layer.forward_routed(x, none, w))


def test_layer_refuses():
    layer = _layer(SHAPES["flat"])
    x = torch.randn(4, 512, device="cuda").bfloat16()
    with pytest.raises(RuntimeError, match="contiguous bf16"):
        layer.forward_routed(x.float(), torch.zeros(4, 2, dtype=torch.int32, device="cuda"), torch.ones(4, 2, device="cuda"))
    with pytest.raises(RuntimeError, match="router_logits"):
        layer.forward(x, torch.zeros(4, 7, device="cuda").bfloat16())
    with pytest.raises(RuntimeError, match="w13"):
        fp8.Fp8MoE(SHAPES["odd"], layer.w13, layer.w13_scale, layer.w2, layer.w2_scale)
    with pytest.raises(RuntimeError, match="top-k"):
        fp8.Fp8MoE(synth.scaled_shape(SHAPES["flat"], act_topk_keep=8), layer.w13, layer.w13_scale, layer.w2, layer.w2_scale)
    assert layer.forward(x[:0], torch.zeros(0, 8, device="cuda").bfloat16()).shape == (0, 512)
