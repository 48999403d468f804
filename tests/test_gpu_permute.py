"""Tokens sorted by expert and back, with weights and gradients, against plain 64-bit forms.

Tolerances: a copy is exact. A sum of k products runs in fp32 (each product and addition off by at most 2^-24 of what it
makes: k + 1 of them on a term) and is rounded once to the output's type, half a step = finfo.eps / 2 of the value (and
half the smallest subnormal, which matters for fp16). A product rounded once is off by half a step and the 2^-24 of fp32.
A dot product's fp32 chain is the terms one thread adds, then 5 steps over the warp and 8 over the warps."""
import pytest
import torch

from tests import fp8_plain as P
from tests import helpers as Hh
from xcaliber_b200 import ops, synth

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]
F32 = 2.0 ** -24


def half_step(t):
    return torch.finfo(t).eps / 2, torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def assert_near(got, ref, tol):
    d = (got.double() - ref).abs()
    assert bool((d <= tol).all()), f"off by {float((d - tol).max()):.3g} more than allowed"


CASES = [  # tokens, experts, k, hidden, dropped
    (1, 8, 2, 4096, 0.0), (1, 1, 1, 1, 0.0), (3, 4, 4, 7, 0.0), (17, 8, 3, 2880, 0.3), (64, 128, 8, 2048, 0.0),
    (33, 16, 9, 136, 0.1), (129, 32, 17, 100, 0.2), (5, 8, 2, 12288, 0.0), (40, 4, 2, 1023, 1.0), (300, 60, 6, 513, 0.05), (21, 8, 2, 2050, 0.0), (9, 8, 8, 4101, 0.1),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,e,k,h,dropped", CASES)
def test_permute_and_its_gradient(n, e, k, h, dropped, dtype):
    row, _, _, r = P.plan(n, e, k, seed=n + h, dropped=dropped)
    x = torch.randn(n, h, device="cuda").to(dtype)
    plan = row.cuda()
    keep = torch.randn(r, h, device="cuda").to(dtype)
    out = ops.permute(x, plan, out=keep.clone())
    want = keep.clone()
    t, s = torch.nonzero(plan >= 0, as_tuple=True)
    want[plan[t, s].long()] = x[t]
    assert torch.equal(out, want)  # rows that no slot names are as they were
    named = torch.zeros(r, dtype=torch.bool, device="cuda")
    named[plan[t, s].long()] = True
    assert torch.equal(ops.permute(x, plan, r), torch.where(named[:, None], want, 0))
    d = torch.randn(r, h, device="cuda").to(dtype)
    d[~named] = float("nan")  # and are not read
    ref, size = P.unpermute(d.nan_to_num(0.0), plan)
    rel, floor = half_step(dtype)
    assert_near(ops.permute_backward(d, plan), ref, rel * ref.abs() + floor + (k + 1) * F32 * size)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("wtype", [None, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,e,k,h,dropped", CASES)
def test_unpermute_and_its_gradients(n, e, k, h, dropped, wtype, dtype):
    row, _, _, r = P.plan(n, e, k, seed=n + h + 1, dropped=dropped)
    plan = row.cuda()
    rows, dy = torch.randn(r, h, device="cuda").to(dtype), torch.randn(n, h, device="cuda").to(dtype)
    w = None if wtype is None else torch.rand(n, k, device="cuda").to(wtype)
    rel, floor = half_step(dtype)
    ref, size = P.unpermute(rows, plan, w)
    y = ops.unpermute(rows, plan, w)
    assert_near(y, ref, rel * ref.abs() + floor + (k + 1) * F32 * size)
    if dropped == 1.0:
        assert not y.any()  # nothing comes back to a token without rows
    keep = torch.randn(r, h, device="cuda").to(dtype)
    drows, dw = ops.unpermute_backward(dy, rows, plan, w, out=keep.clone())
    t, s = torch.nonzero(plan >= 0, as_tuple=True)
    at = plan[t, s].long()
    want, tol = keep.double(), torch.zeros_like(keep, dtype=torch.float64)
    want[at] = dy.double()[t] * (1.0 if w is None else w.double()[t, s][:, None])
    tol[at] = (rel + F32) * want[at].abs() + floor
    assert_near(drows, want, tol)
    assert dw.dtype == torch.float32
    prod = torch.zeros(n, k, h, dtype=torch.float64, device="cuda")
    prod[t, s] = dy.double()[t] * rows.double()[at]
    chain = -(-h // 256) + 16 + 14
    assert_near(dw, prod.sum(-1), chain * F32 * prod.abs().sum(-1))
    assert not dw[plan < 0].any()


def test_autograd_against_formula_and_differences():
    """y = unpermute(permute(x) * c, w): the gradients are the formulas', and the slope of the loss along a direction. The
    loss is linear in x and in w, so a difference of any width is the slope up to fp32: with terms of size 1, N * k * H =
    9600 of them, 9600 * 2^-24 per unit of width bounds what rounding does; a bound of 2e-3 on sums of that size holds it."""
    torch.manual_seed(0)
    n, e, k, h = 40, 8, 3, 80
    row, _, _, r = P.plan(n, e, k, seed=3, dropped=0.1)
    plan = row.cuda()
    x = torch.randn(n, h, device="cuda", requires_grad=True)
    w = torch.rand(n, k, device="cuda", requires_grad=True)
    c, dy = torch.randn(r, h, device="cuda"), torch.randn(n, h, device="cuda")

    def loss(x, w):
        return (ops.unpermute(ops.permute(x, plan, r) * c, plan, w).double() * dy).sum()

    gx, gw = torch.autograd.grad(loss(x, w), (x, w))
    ok = (plan >= 0)[..., None]
    ct = c.double()[plan.clamp_min(0).long()] * ok
    xd, wd = x.detach().double(), w.detach().double()
    # three terms below 32 each, five roundings of 2^-24 on each; a chain of 31 additions on sums of magnitudes below 512
    assert_near(gx, (ct * wd[..., None] * dy.double()[:, None]).sum(1), 1e-4)
    assert_near(gw, (ct * xd[:, None] * dy.double()[:, None]).sum(-1), 1e-3)
    vx, vw = torch.randn_like(x), torch.randn_like(w)
    with torch.no_grad():
        assert abs(float((loss(x + vx, w) - loss(x - vx, w)) / 2 - (gx.double() * vx).sum())) < 2e-3
        assert abs(float((loss(x, w + vw) - loss(x, w - vw)) / 2 - (gw.double() * vw).sum())) < 2e-3


def test_route_pack_is_the_layers_permutation_and_drops_slots():
    torch.manual_seed(1)
    n, e, k = 700, 16, 2
    idx = torch.stack([torch.randperm(e)[:k] for _ in range(n)]).to(torch.int32)
    idx[::7, 1] = -1
    w = torch.rand(n, k).to(torch.bfloat16)
    r = ops.route_pack(idx.cuda(), w.cuda(), e, num_shared=1)
    assert int(r.status[0]) == 0
    counts = torch.bincount(idx[idx >= 0].long(), minlength=e).tolist() + [n]
    assert r.counts.tolist() == counts
    assert r.offsets.tolist() == [sum(-(-c // 128) * 128 for c in counts[:i]) for i in range(e + 2)]
    row = r.topk_row.cpu()
    assert bool((row[:, :k][idx < 0] == -1).all()) and row[row >= 0].unique().numel() == int((row >= 0).sum())
    for s in range(k + 1):
        for t in (0, 1, 6, 7, 350, n - 1):
            if row[t, s] >= 0:
                ex = e if s == k else int(idx[t, s])
                assert r.offsets[ex] <= row[t, s] < r.offsets[ex] + r.counts[ex] and int(r.row_token[row[t, s]]) == t
    assert bool((r.topk_w[:, k] == 1).all()) and r.rows_in_use == n * (k + 1) and int(r.offsets[-1]) <= r.num_rows


@pytest.mark.parametrize("n", [1, 40, 700])  # one and several chunks of the kernel
def test_route_pack_gives_every_slot_a_row_of_its_own(n):
    """An expert named in several slots of a token: as many rows, in slot order, behind those of the tokens before."""
    g = torch.Generator().manual_seed(n)
    e, k = 4, 6
    idx = torch.randint(-1, e, (n, k), generator=g, dtype=torch.int32)
    idx[0] = 2
    r = ops.route_pack(idx.cuda(), torch.rand(n, k, generator=g).bfloat16().cuda(), e)
    assert int(r.status[0]) == 0 and r.counts.tolist() == [int((idx == x).sum()) for x in range(e)]
    want = torch.full((n, k), -1, dtype=torch.int32)
    for x in range(e):
        t, s = torch.nonzero(idx == x, as_tuple=True)  # token by token, slot by slot
        want[t, s] = int(r.offsets[x]) + torch.arange(len(t), dtype=torch.int32)
        assert torch.equal(r.row_token.cpu()[int(r.offsets[x]):int(r.offsets[x]) + len(t)], t.int())
    assert torch.equal(r.topk_row.cpu(), want)


def _route_kernels(call):
    """Names of the route pack's kernels that a call launches."""
    from torch.profiler import ProfilerActivity, profile

    call()
    torch.cuda.synchronize()
    with profile(activities=[ProfilerActivity.CUDA]) as p:
        call()
        torch.cuda.synchronize()
    names = [e.name for e in p.events()]
    if not names:
        pytest.skip("the profiler sees no kernels here")
    return [n for n in names if "route_scatter_kernel" in n]


@pytest.mark.parametrize("n", [9, 300])
def test_only_routing_of_a_caller_is_checked_for_an_expert_twice(n):
    """The check costs time: the router's output (of the gated forward too) and a single slot per token go without it."""
    shape = synth.SHAPES["toy"]
    w, layer = Hh.build_layer(shape)
    x, logits = (t.cuda() for t in synth.make_inputs(shape, w, n))
    gate = w.router_weight.to(torch.bfloat16).cuda()
    idx, wt = ops.router_topk(logits, shape)
    unchecked = [lambda: layer.forward_gated(x, gate), lambda: ops.route_pack(idx[:, :1], wt[:, :1], shape.num_experts)]
    if n > 32:  # smaller batches have a kernel of their own for the whole front
        unchecked.append(lambda: layer.forward(x, logits))
    for call in unchecked:
        names = _route_kernels(call)
        assert len(names) == 1 and "<false>" in names[0]
    for call in (lambda: layer.forward_routed(x, idx, wt), lambda: ops.route_pack(idx, wt, shape.num_experts)):
        names = _route_kernels(call)
        assert len(names) == 1 and "<true>" in names[0]


def test_plan_strides_rows_outside_streams_and_empty_calls():
    n, k, h = 50, 2, 256
    row, _, _, r = P.plan(n, 8, k, seed=5)
    wide = torch.full((n, 5), -1, dtype=torch.int32, device="cuda")
    wide[:, :k] = row.cuda()
    x = torch.randn(n, h, device="cuda", dtype=torch.bfloat16)
    ref = ops.permute(x, row.cuda(), r)
    assert torch.equal(ops.permute(x, wide[:, :k], r), ref)
    assert torch.equal(ops.permute(x, wide, r), ref)
    far = wide.clone()
    far[:, 2:] = torch.tensor([r, r + 1000, 2 ** 31 - 1], dtype=torch.int32, device="cuda")  # rows that are not there
    assert torch.equal(ops.permute(x, far, r), ref)
    w = torch.rand(n, 5, device="cuda")
    assert torch.equal(ops.unpermute(ref, far, w), ops.unpermute(ref, wide[:, :k], w[:, :k]))
    assert not ops.unpermute_backward(x, ref, far, w)[1][:, 2:].any()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        on_s = ops.unpermute(ops.permute(x, wide, r), wide, w)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(on_s, ops.unpermute(ref, wide, w))
    none = torch.empty(0, k, dtype=torch.int32, device="cuda")
    assert ops.permute(x[:0], none, 128).shape == (128, h) and not ops.permute(x[:0], none, 128).any()
    assert ops.unpermute(ref, none).shape == (0, h)
    no_slot = torch.empty(n, 0, dtype=torch.int32, device="cuda")
    assert not ops.unpermute(ref, no_slot).any()
    assert not ops.unpermute(ref[:0], row.cuda()).any()
    assert ops.unpermute_backward(x, ref, no_slot)[1].shape == (n, 0)


def test_gradients_in_a_captured_graph():
    """Forward and both gradients captured (through autograd, the leaves having been used eagerly first) and replayed on
    other inputs give what the eager calls give."""
    n, k, h = 33, 4, 512
    row, _, _, r = P.plan(n, 8, k, seed=6)
    plan = row.cuda()

    def step(x, w, dy):
        y = ops.unpermute(ops.permute(x, plan, r), plan, w)
        return (y.detach(), *torch.autograd.grad(y, (x, w), dy))

    def inputs(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        return (torch.randn(n, h, device="cuda", generator=g).bfloat16(), torch.rand(n, k, device="cuda", generator=g),
                torch.randn(n, h, device="cuda", generator=g).bfloat16())

    fixed = inputs(0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(fixed[0].requires_grad_(), fixed[1].requires_grad_(), fixed[2])
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*fixed)
    for seed in (1, 2):
        new = inputs(seed)
        with torch.no_grad():
            for a, b in zip(fixed, new):
                a.copy_(b)
        graph.replay()
        want = step(new[0].requires_grad_(), new[1].requires_grad_(), new[2])
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("what", ["plan type", "plan shape", "plan device", "strides", "type", "width", "weights shape", "weights type"])
def test_refusals(what):
    row, _, _, r = P.plan(6, 4, 2, seed=1)
    plan = row.cuda()
    rows, w, y = torch.randn(r, 64, device="cuda"), torch.rand(6, 2, device="cuda"), torch.empty(6, 64, device="cuda")
    if what == "plan type":
        plan = plan.long()
    elif what == "plan shape":
        plan = plan[:5]
    elif what == "plan device":
        plan = row
    elif what == "strides":
        rows = torch.randn(r, 128, device="cuda")[:, ::2]
    elif what == "type":
        rows = rows.double()
    elif what == "width":
        rows = rows[:, :32].contiguous()
    elif what == "weights shape":
        w = w[:, :1]
    else:
        w = w.half()
    with pytest.raises(RuntimeError):
        ops.unpermute(rows, plan, w, out=y)
    with pytest.raises(RuntimeError):
        ops.unpermute_backward(y, rows, plan, w)
    if not what.startswith("weights"):
        with pytest.raises(RuntimeError):
            ops.permute(y, plan, out=rows)
