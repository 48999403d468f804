"""Refusals of the operators around FP8 experts, and the plain forms the GPU tests compare with: no GPU needed."""
import ctypes as C
import re
from pathlib import Path

import pytest
import torch

from tests import fp8_plain as P
from xcaliber_b200 import _lib, fp8, ops, synth

A = 1 << 20  # an aligned address that no refused call may touch
ARG, SHAPE, LIMIT = 1, 2, 6


@pytest.mark.parametrize("args,rc", [
    ((A, A, -1, 64, 2, 2, 128, 0, A, None), ARG), ((None, A, 4, 64, 2, 2, 128, 0, A, None), ARG),
    ((A, None, 4, 64, 2, 2, 128, 0, A, None), ARG), ((A, A, 4, 64, 2, 2, 128, 0, None, None), ARG),
    ((A, A, 4, 0, 2, 2, 128, 0, A, None), SHAPE), ((A, A, 4, 64, 2, 1, 128, 0, A, None), SHAPE),
    ((A, A, 4, 64, 2, 2, 128, 3, A, None), SHAPE), ((A, A, 4, 64, 2, 2, -1, 0, A, None), ARG),
    ((None, None, 0, 64, 2, 2, 128, 0, None, None), 0), ((A, A, 4, 64, 2, 2, 0, 0, None, None), 0),
])
def test_permute_refuses(built_lib, args, rc):
    assert built_lib.xmoe_permute(*args) == rc


@pytest.mark.parametrize("args,rc", [
    ((A, A, A, 1, 2, 4, 64, 2, 2, 128, 0, A, None), SHAPE),  # weights of fp16
    ((A, A, A, 0, 1, 4, 64, 2, 2, 128, 0, A, None), SHAPE),  # weights' rows shorter than k
    ((A, A, None, 0, 0, 4, 64, 2, 2, 128, 9, A, None), SHAPE), ((None, A, None, 0, 0, 4, 64, 2, 2, 128, 0, A, None), ARG),
    ((A, A, None, 0, 0, 4, 64, 2, 2, 128, 0, None, None), ARG), ((A, A, None, 0, 0, 0, 64, 2, 2, 128, 0, None, None), 0),
])
def test_unpermute_refuses(built_lib, args, rc):
    assert built_lib.xmoe_unpermute(*args) == rc


@pytest.mark.parametrize("drows,dw,rc", [(None, A, ARG), (A, None, ARG), (2 * A, A, ARG)])
def test_unpermute_backward_refuses(built_lib, drows, dw, rc):
    # rows at 2 * A: drows may not be the same buffer
    assert built_lib.xmoe_unpermute_backward(A, 2 * A, A, None, 0, 0, 4, 64, 2, 2, 128, 0, drows, dw, None) == rc


@pytest.mark.parametrize("args,rc", [
    ((A, 0, 4, 64, 32, None, 0, 0, 0, A, 64, A, 4, None), SHAPE),    # rows overlap
    ((A, 0, 4, 64, 64, None, 0, 0, 0, A, 72, A, 4, None), SHAPE),    # code rows not at multiples of 16
    ((A, 0, 4, 64, 64, None, 0, 0, 0, A, 64, A, 3, None), SHAPE),    # scales shorter than the rows
    ((A, 0, 4, 64, 64, None, 0, 0, 0, A + 8, 64, A, 4, None), SHAPE),
    ((A, 5, 4, 64, 64, None, 0, 0, 0, A, 64, A, 4, None), SHAPE), ((A, 0, -4, 64, 64, None, 0, 0, 0, A, 64, A, 4, None), ARG),
    ((A, 0, 4, 64, 64, A, 2, 1, 128, A, 64, A, 128, None), SHAPE),   # plan's rows shorter than k
    ((A, 0, 4, 64, 64, A, 2, 2, 128, A, 64, A, 124, None), SHAPE), ((A, 0, 4, 64, 64, A, 2, 2, -1, A, 64, A, 128, None), ARG),
    ((None, 0, 0, 64, 64, None, 0, 0, 0, None, 64, None, 0, None), 0),
])
def test_quant_refuses(built_lib, args, rc):
    assert built_lib.xmoe_fp8_quant(*args) == rc


def test_glu_and_weight_quant_refuse(built_lib):
    lib = built_lib
    ok = (A, 0, 8, 64, 0, 1.0, 1.0, None, None, 0, A, 64, A, 8, None)

    def glu(**kw):
        names = "h dtype rows inter act alpha limit counts offsets mats q ldq scale lds stream".split()
        return lib.xmoe_glu_fp8_quant(*{**dict(zip(names, ok)), **kw}.values())

    assert glu(rows=-1) == ARG and glu(act=3) == SHAPE and glu(ldq=48) == SHAPE and glu(lds=4) == SHAPE
    assert glu(counts=A) == ARG and glu(counts=A, offsets=A, mats=2000) == LIMIT and glu(h=None) == ARG
    assert glu(rows=0, lds=0) == 0
    assert lib.xmoe_glu_backward(A, A, 0, 8, 64, 0, 1.0, 1.0, None, None, 0, A, None) == ARG  # in place
    assert lib.xmoe_glu_backward(A, A, 0, 8, 0, 0, 1.0, 1.0, None, None, 0, 2 * A, None) == SHAPE
    assert lib.xmoe_fp8_quant_weight(A, 0, 1, 64, 64, A, 32, A, None) == SHAPE
    assert lib.xmoe_fp8_quant_weight(A, 0, 1, 64, 64, None, 64, A, None) == ARG
    assert lib.xmoe_fp8_quant_weight(A, 0, 0, 64, 64, None, 64, None, None) == 0


@pytest.mark.parametrize("off", [1, 4, 8])
def test_weight_quant_refuses_codes_off_16_bytes(built_lib, off):
    # codes are stored eight at a time, and the products' copies want rows at multiples of 16 bytes
    assert built_lib.xmoe_fp8_quant_weight(A, 0, 1, 64, 64, A + off, 64, A, None) == SHAPE


def test_products_refuse(built_lib):
    lib = built_lib
    names = "x ldx xs lds w ldw wmat ws counts offsets mats rows used n k tr out odt ldo stream".split()
    ok = dict(zip(names, (A, 128, A, 8, A, 128, 256 * 128, A, A, A, 2, 8, 0, 256, 128, 0, A, 0, 256, None)))

    def grouped(**kw):
        return lib.xmoe_fp8_grouped_gemm(*{**ok, **kw}.values())

    assert grouped(ldx=112) == SHAPE and grouped(ldx=136) == SHAPE and grouped(ldw=120) == SHAPE and grouped(lds=4) == SHAPE
    assert grouped(lds=10) == SHAPE and grouped(ldo=128) == SHAPE and grouped(wmat=128) == SHAPE
    assert grouped(wmat=256 * 128 + 8) == SHAPE and grouped(odt=3) == SHAPE and grouped(n=0) == SHAPE and grouped(mats=0) == SHAPE
    assert grouped(mats=2000) == LIMIT and grouped(rows=-1) == ARG and grouped(used=-1) == ARG and grouped(x=None) == ARG
    assert grouped(counts=None) == ARG and grouped(xs=A + 4) == SHAPE and grouped(out=None) == ARG
    assert grouped(tr=1) == SHAPE  # contracts over n = 256: x is too narrow
    assert grouped(rows=0, lds=0) == 0
    assert lib.xmoe_fp8_gemm(A, 120, A, 8, A, 128, A, 8, 256, 128, 0, A, 0, 256, None) == SHAPE
    assert lib.xmoe_fp8_status(None, None) == ARG


TOP = 2 ** 31 - 16  # fits 32 bits; a kernel that rounds it up to its next step does not


def test_sizes_at_the_end_of_32_bits_are_refused(built_lib):
    """Kernels step through rows and columns in 32 bits, past the last by up to a block or a CTA's share."""
    lib = built_lib
    assert lib.xmoe_permute(A, A, 4, TOP, 2, 2, 128, 2, A, None) == LIMIT
    assert lib.xmoe_unpermute_backward(A, 2 * A, A, None, 0, 0, 1, TOP, 2, 2, 1, 2, 4 * A, A, None) == LIMIT
    assert lib.xmoe_unpermute(A, A, None, 0, 0, 1, 64, TOP, TOP, 128, 0, A, None) == LIMIT
    assert lib.xmoe_fp8_quant(A, 0, TOP, 1, 1, None, 0, 0, 0, A, 16, A, TOP, None) == LIMIT
    assert lib.xmoe_fp8_quant(A, 0, 1, TOP, TOP, None, 0, 0, 0, A, TOP, A, 4, None) == LIMIT
    assert lib.xmoe_fp8_quant(A, 0, 1, 64, 64, A, TOP, TOP, 128, A, 64, A, 128, None) == LIMIT
    assert lib.xmoe_fp8_quant_weight(A, 0, 1, TOP, 1, A, 16, A, None) == LIMIT
    assert lib.xmoe_fp8_quant_weight(A, 0, 1, 1, TOP, A, TOP, A, None) == LIMIT
    assert lib.xmoe_glu_fp8_quant(A, 0, TOP, 1, 0, 1.0, 1.0, None, None, 0, A, 16, A, TOP, None) == LIMIT
    assert lib.xmoe_glu_backward(A, A, 0, TOP, 1, 0, 1.0, 1.0, None, None, 0, 2 * A, None) == LIMIT
    for rows, n, k in ((TOP, 1, 16), (1, TOP, 16), (1, 16, TOP)):
        assert lib.xmoe_fp8_gemm(A, max(k, 16), A, max(rows, 4), A, max(k, 16), A, rows, n, k, 0, A, 0, n, None) == LIMIT


@pytest.mark.parametrize("n,e,k,shared,rc", [(2 ** 26, 8, 32, 0, LIMIT), (2 ** 31 - 1, 8, 1, 0, LIMIT), (2 ** 27 - 1, 512, 16, 0, LIMIT),
                                             (4, -1, 2, 2, SHAPE), (4, 8, 2, -1, SHAPE), (4, 8, -1, 2, SHAPE)])
def test_route_pack_refuses(built_lib, n, e, k, shared, rc):
    """Row numbers are 32-bit, padding of the experts' segments included."""
    assert built_lib.xmoe_route_pack(A, A, n, e, k, max(k + shared, 8), shared, A, A, A, A, A, A, A, A, None) == rc


def test_epilogue_warps_give_up_together():
    """No lane of an epilogue warp leaves the walk over a tile's blocks by itself, where a shuffle or an aligned tensor-memory
    read of the whole warp follows; the warp decides behind the walk. (A wait that runs out is not provoked on a GPU; the
    epilogue sections of the products are read instead.)"""
    source = (Path(_lib.__file__).parent / "csrc" / "fp8_gemm.cu").read_text()
    sections = re.findall(r"const int q = warp & 3, part = .*?\n    __syncthreads\(\);", source, re.S)
    assert len(sections) == 2  # both kernels
    for text in sections:
        walk, behind = re.search(r"\n( +)for \(int kb = .*?\n\1\}\n(.*)", text, re.S).group(0, 2)
        walk = walk[:-len(behind)]
        voted, own = len(re.findall(r"!mbar_wait_warp\(", walk)), walk.count("ok &= mbar_wait(")
        assert voted + own == 2 and len(re.findall(r"\bmbar_wait\w*\(", walk)) == 2
        assert len(re.findall(r"\b(?:break|return|continue|goto)\b", walk)) == voted
        assert not own or behind.lstrip().startswith("ok = __all_sync(0xffffffffu, ok);")


def test_python_refuses_what_it_cannot_do():
    x = torch.zeros(4, 64)
    plan = torch.zeros(4, 2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="num_rows or out"):
        ops.permute(x, plan)
    with pytest.raises(RuntimeError, match="not differentiable"):
        ops.permute(x.clone().requires_grad_(), plan, out=torch.zeros(128, 64))
    with pytest.raises(RuntimeError, match="not differentiable"):
        ops.unpermute(x.clone().requires_grad_(), plan, out=torch.zeros(4, 64))
    with pytest.raises(RuntimeError, match="num_rows or out"):
        fp8.quant(x, plan)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.route_pack(plan, plan.bfloat16(), 8)
    with pytest.raises(NotImplementedError):  # no CPU kernel, no fallback
        fp8.matmul(x.to(torch.float8_e4m3fn), torch.ones(4, 1), x.to(torch.float8_e4m3fn), torch.ones(1, 1))


def calls_into_out(dev):
    """Every call that writes into tensors of the caller: (name, the tensors, the call)."""
    n, k, h, r = 4, 2, 64, 128
    x, rows, plan = torch.zeros(n, h, device=dev), torch.zeros(r, h, device=dev), torch.arange(n * k, dtype=torch.int32).view(n, k).to(dev)
    w = torch.ones(n, k, device=dev)
    codes = torch.zeros(n, h, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
    scale = fp8.empty_rows(n, h, dev)[1].zero_()
    mats = torch.zeros(1, h, h, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
    ws = torch.ones(1, 1, 1, device=dev)
    counts, offsets = torch.tensor([n], dtype=torch.int32).to(dev), torch.tensor([0, 128], dtype=torch.int32).to(dev)
    two = torch.zeros(n, 2 * h, device=dev)
    q = [fp8.empty_rows(m, h, dev) for m in (n, r, n)]
    y, drows, dh = torch.zeros(n, h, device=dev), torch.zeros(r, h, device=dev), torch.zeros(n, 2 * h, device=dev)
    a, b = torch.zeros(n, h, device=dev), torch.zeros(n, h, device=dev)
    return [("permute", [rows], lambda: ops.permute(x, plan, out=rows)),
            ("unpermute", [y], lambda: ops.unpermute(drows.clone(), plan, w, out=y)),
            ("unpermute_backward", [drows], lambda: ops.unpermute_backward(x, rows, plan, w, out=drows)),
            ("quant", list(q[0]), lambda: fp8.quant(x, out=q[0])), ("quant sorted", list(q[1]), lambda: fp8.quant(x, plan, out=q[1])),
            ("glu_quant", list(q[2]), lambda: fp8.glu_quant(two, out=q[2])),
            ("glu_backward", [dh], lambda: fp8.glu_backward(x, two, out=dh)),
            ("matmul", [a], lambda: fp8.matmul(codes, scale, mats[0], ws[0], out=a)),
            ("grouped_matmul", [b], lambda: fp8.grouped_matmul(codes, scale, mats, ws, counts, offsets, out=b))]


def assert_writes_are_seen(dev):
    for name, outs, call in calls_into_out(dev):
        before = [t._version for t in outs]
        call()
        assert all(t._version > v for t, v in zip(outs, before)), name
    leaf = torch.zeros(128, 64, device=dev, requires_grad=True)
    _, (rows,), call = calls_into_out(dev)[0]
    loss = (leaf * rows).sum()  # keeps rows for the gradient
    call()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_autograd_sees_writes_into_out():
    """A tensor of the caller counts as changed by a call that writes into it: a backward pass through a value saved before
    the write is refused, as after torch's own in-place operations."""
    assert_writes_are_seen("meta")


def test_out_that_requires_gradients_is_refused():
    """No call into `out` is recorded for a gradient: a leaf, or a value of an eager graph, is not overwritten in silence."""
    for k, (name, outs, _) in enumerate(calls_into_out("meta")):
        for i in range(len(outs)):
            _, outs, call = calls_into_out("meta")[k]
            if outs[i].dtype == torch.float8_e4m3fn:
                continue
            outs[i].requires_grad_()
            with pytest.raises(RuntimeError, match="not differentiable"):
                call()
            with torch.no_grad():
                call()


def _cpu_layer(**kw):
    shape = synth.MoEShape("fp8_small", 128, 64, 4, 2, **kw)
    codes = lambda *d: torch.zeros(*d, dtype=torch.uint8).view(torch.float8_e4m3fn)  # noqa: E731
    return shape, (codes(4, 128, 128), torch.ones(4, 1, 1), codes(4, 128, 64), torch.ones(4, 1, 1))


def test_layer_refuses_tensors_of_other_devices():
    """Before anything is launched: a kernel would follow the address of another device, or of the host."""
    shape, weights = _cpu_layer()
    layer = fp8.Fp8MoE(shape, *weights)
    x = torch.zeros(4, 128, dtype=torch.bfloat16)
    logits, idx, w = torch.zeros(4, 4, dtype=torch.bfloat16), torch.zeros(4, 2, dtype=torch.int32), torch.ones(4, 2)
    for xd in (x, x.to("meta")):
        with pytest.raises(RuntimeError, match="x must be .* on the device of the weights"):
            layer.forward(xd, logits)
        with pytest.raises(RuntimeError, match="x must be .* on the device of the weights"):
            layer.forward_routed(xd, idx, w)
    layer.w13 = layer.w13.to("meta")  # stands for a CUDA device
    with pytest.raises(RuntimeError, match="router_logits must be .* on x's device"):
        layer._check_logits(x.to("meta"), logits)


def test_layer_refuses_a_bias_that_is_not_one_per_expert():
    shape, weights = _cpu_layer(scoring="sigmoid", router_bias=True)
    for bias in (torch.zeros(3), torch.zeros(8), torch.zeros(4, 1), torch.zeros(())):
        with pytest.raises(RuntimeError, match="router_bias must be"):
            fp8.Fp8MoE(shape, *weights, bias)


def test_layout_of_empty_rows():
    codes, scale = fp8.empty_rows(5, 130, "cpu")
    assert codes.shape == (5, 130) and codes.stride() == (144, 1) and codes.dtype == torch.float8_e4m3fn
    assert scale.shape == (5, 2) and scale.stride() == (1, 8)


def test_plain_rounding_is_the_formats():
    """e4m3_round against torch's own conversion, on every value, every midpoint and its fp32 neighbours."""
    v = P.e4m3_values()
    mid = ((v[1:] + v[:-1]) / 2).float()
    all_of = torch.cat([v.float(), mid, mid.nextafter(torch.tensor(1e9)), mid.nextafter(torch.tensor(0.0))])
    all_of = torch.cat([all_of, -all_of])
    assert torch.equal(P.e4m3_round(all_of.double()), all_of.to(torch.float8_e4m3fn).double())


def test_ctypes_signatures_of_the_new_calls(built_lib):
    for name in ("xmoe_permute", "xmoe_fp8_grouped_gemm", "xmoe_fp8_status"):
        assert name in _lib.SIGNATURES and getattr(built_lib, name).restype is C.c_int
