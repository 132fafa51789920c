"""GPU checks of the router, the token plan and the movement of tokens
(``kernels.moe_route``, ``token_plan``, ``moe_dispatch``, ``moe_combine``)
against their definitions in 64 bits.

Ids, plans and copies are exact.  Gate weights and losses are f32 sums of up to
E (losses: T) positive terms, each within a few roundings: a relative error of
(E + 64) 2^-24 for the weights, (T + E + 64) 2^-24 for the losses, plus, through
the exponent, 2^-24 times the largest logit's magnitude.  A result of the
tensors' own type adds one rounding of that type.
"""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
HALF_ULP = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -24}      # relative, 8 / 11 / 24 bits
TINY = {BF16: 2.0 ** -134, F16: 2.0 ** -25, F32: 2.0 ** -150}     # half of the smallest step


def _rand(shape, seed, dtype=F32, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def _close(got, want, bound, what):
    """|got - want| <= bound elementwise, bound already per element."""
    bad = (got.double() - want).abs() > bound
    assert not bad.any(), (what, int(bad.sum()), float((got.double() - want).abs().max()))


# --- plan -------------------------------------------------------------------


def _plan_ref(ids, E, multiple):
    """rows, src, counts, offs by their definition (numpy, entry by entry)."""
    flat = np.asarray(ids).reshape(-1)
    n = flat.size
    counts = np.array([(flat == e).sum() for e in range(E)], np.int64)
    sizes = -(-counts // multiple) * multiple
    ends = np.cumsum(sizes)
    rows = np.full(n, -1, np.int64)
    M = (n + min(E, n) * (multiple - 1)) // multiple * multiple
    src = np.full(M, -1, np.int64)
    for e in range(E):
        at = np.nonzero(flat == e)[0]
        rows[at] = ends[e] - sizes[e] + np.arange(at.size)
        src[rows[at]] = at
    return rows.reshape(np.shape(ids)), src, counts, ends


def _check_plan(plan, ids, E, multiple):
    rows, src, counts, ends = _plan_ref(ids, E, multiple)
    for name, got, want in (("rows", plan.rows, rows), ("src", plan.src, src), ("counts", plan.counts, counts),
                            ("offs", plan.offs, ends)):
        assert got.dtype == torch.int32
        np.testing.assert_array_equal(got.cpu().numpy().reshape(want.shape), want, err_msg=name)


@pytest.mark.parametrize("T,k,E,multiple", [
    (0, 2, 4, 32), (1, 1, 1, 1), (1, 4, 32, 32), (63, 1, 5, 1), (64, 2, 8, 32), (65, 3, 3, 7), (1000, 1, 64, 1),
    (1024, 1, 65, 16), (1025, 1, 300, 32), (4097, 5, 37, 32), (700, 8, 1024, 32), (20011, 2, 1000, 4), (70000, 8, 9, 128),
])
def test_token_plan(gpu, T, k, E, multiple):
    import kernels
    ids = np.random.default_rng(T + E).integers(-2, E + 2, (T, k))       # ids outside the groups among them
    for dtype in (torch.int32, torch.int64):
        plan = kernels.token_plan(torch.tensor(ids, dtype=dtype, device=gpu), E, multiple)
        _check_plan(plan, ids, E, multiple)


def test_token_plan_one_group_and_flat_ids(gpu):
    """All entries in one group, or in none; (T,) ids; ids that are a strided view."""
    import kernels
    for fill in (3, -1):
        ids = np.full((3000,), fill)
        plan = kernels.token_plan(torch.tensor(ids, device=gpu), 8, 32)
        assert tuple(plan.rows.shape) == (3000, 1)
        _check_plan(plan, ids.reshape(-1, 1), 8, 32)
    wide = torch.randint(0, 8, (500, 4), device=gpu, dtype=torch.int32)
    _check_plan(kernels.token_plan(wide[:, 1], 8, 1), wide[:, 1:2].cpu().numpy(), 8, 1)
    huge = torch.tensor([0, 1 << 40, -(1 << 40), 2], device=gpu)          # outside 32 bits: no group
    _check_plan(kernels.token_plan(huge, 4, 1), np.array([[0], [-1], [-1], [2]]), 4, 1)


# --- router -----------------------------------------------------------------


def _route_ref(logits, k, normalize, gw=None, gb=0.0, gz=0.0):
    """The router in 64 bits: (weights, ids, balance, z, gradient of logits)."""
    l = logits.double().detach().requires_grad_()
    T, E = l.shape
    live = (l > float("-inf")).any(dim=1)
    safe = torch.where(live.unsqueeze(1), l, 0.0)
    p = torch.where(live.unsqueeze(1), torch.softmax(safe, dim=1), 0.0)
    lse = torch.where(live, torch.logsumexp(safe, dim=1), 0.0)
    order = torch.argsort(l.detach(), dim=1, descending=True, stable=True)[:, :k]
    open_ = l.detach().gather(1, order) > float("-inf")
    raw = torch.where(open_, p.gather(1, order), 0.0)
    w = raw / torch.where(live, raw.sum(dim=1), 1.0).unsqueeze(1) if normalize else raw
    ids = torch.where(open_, order, -1)
    counts = torch.stack([(ids == e).sum() for e in range(E)]).double()
    n = max(1, int(live.sum()))
    balance = E * (counts / (n * k) * (p.sum(dim=0) / n)).sum()
    z = (lse ** 2).sum() / n
    total = balance * gb + z * gz
    if gw is not None:
        total = total + (w * gw.double()).sum()
    if T:
        total.backward()
    return w.detach(), ids, balance.detach(), z.detach(), l.grad


def _check_route(logits, k, normalize, seed=0, multiple=32):
    import kernels
    T, E = logits.shape
    gw, gb, gz = _rand((T, k), seed + 1), 0.7, 0.3
    x = logits.detach().clone().requires_grad_()
    r = kernels.moe_route(x, k, normalize=normalize, multiple_of=multiple)
    w, ids, balance, z, grad = _route_ref(logits, k, normalize, gw, gb, gz)
    assert r.weights.dtype == F32 and r.ids.dtype == torch.int32
    assert torch.equal(r.ids.long(), ids)
    _check_plan(r.plan, ids.cpu().numpy(), E, multiple)
    finite = logits.double()[torch.isfinite(logits)]
    top = float(finite.abs().max()) if finite.numel() else 0.0
    ew = (E + 64 + 4 * top) * 2.0 ** -24
    el = (T + E + 64 + 4 * top) * 2.0 ** -24
    _close(r.weights, w, ew * w + 2.0 ** -126, "weights")
    _close(r.balance_loss, balance, el * balance, "balance")
    _close(r.z_loss, z, el * (z + 1), "z")
    torch.autograd.backward((r.weights, r.balance_loss, r.z_loss),
                            (gw, torch.tensor(gb, device="cuda"), torch.tensor(gz, device="cuda")))
    assert x.grad.dtype == logits.dtype
    # terms of a gradient: gates (at most 2 |gw| each, k of them and their mean), balance and z
    if T:
        size = 2 * gw.double().abs().sum(dim=1, keepdim=True) + gb * E + 2 * gz * (top + 6)
        _close(x.grad, grad, HALF_ULP[logits.dtype] * grad.abs() * 1.01 + 4 * ew * size + TINY[logits.dtype], "grad")
    # the same without gradients, bit for bit
    with torch.no_grad():
        q = kernels.moe_route(x, k, normalize=normalize, multiple_of=multiple)
    for a, b in ((r.weights, q.weights), (r.ids, q.ids), (r.balance_loss, q.balance_loss), (r.z_loss, q.z_loss),
                 (r.plan.rows, q.plan.rows)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("T,E,k,dtype", [
    (0, 8, 2, F32), (1, 1, 1, F32), (1, 32, 4, BF16), (2, 2, 2, F16), (63, 8, 3, F32), (64, 9, 9, BF16), (65, 16, 16, F32),
    (257, 17, 5, F16), (1000, 64, 32, F32), (513, 65, 8, BF16), (300, 128, 8, F32), (255, 200, 6, F16), (129, 257, 8, F32),
    (70, 512, 32, BF16), (9000, 256, 8, BF16), (40000, 3, 2, F32), (17000, 8, 2, BF16),
])
def test_moe_route(gpu, T, E, k, dtype, normalize):
    _check_route(_rand((T, E), T + E, dtype, 2.0), k, normalize, seed=T)


@pytest.mark.parametrize("T,E,k", [(40000, 64, 4), (33000, 33, 3), (16385, 64, 1), (16640, 32, 4)])
def test_moe_route_and_plan_of_many_workgroups(gpu, T, E, k):
    """Tables of workgroup counts on both sides of the size up to which every
    workgroup adds them up itself."""
    import kernels
    _check_route(_rand((T, E), T + E, BF16, 2.0), k, True, seed=T)
    ids = np.random.default_rng(T).integers(-1, E, (T, k))
    _check_plan(kernels.token_plan(torch.tensor(ids, device=gpu), E, 32), ids, E, 32)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_moe_route_masks(gpu, dtype):
    """Closed experts, rows with fewer open experts than choices, rows with none,
    masks of the type's lowest value, equal logits, zeros of both signs."""
    x = _rand((400, 24), 5, dtype, 1.5)
    x[torch.rand((400, 24), generator=torch.Generator("cuda").manual_seed(1), device="cuda") < 0.5] = float("-inf")
    x[50:60] = float("-inf")                    # no expert
    x[60:70] = float("-inf")
    x[60:70, 7] = 1.0                           # one expert
    x[70:80, 3:] = float("-inf")                # three
    x[80:90] = 0.25                             # all equal: the lowest experts
    x[90:100] = 0.0
    x[90:100, ::2] = -0.0
    x[390:] = float("-inf")                     # padding at the end
    for normalize in (True, False):
        _check_route(x, 6, normalize)
    low = x.clone()
    low[low == float("-inf")] = torch.finfo(dtype).min      # a finite mask: every row has its choices
    import kernels
    r = kernels.moe_route(low, 6)
    _, ids, _, _, _ = _route_ref(low, 6, True)
    assert torch.equal(r.ids.long(), ids)
    assert torch.isfinite(r.weights).all() and torch.isfinite(r.balance_loss)
    _close(r.weights[50:60], torch.full((10, 6), 1 / 6, device=gpu, dtype=torch.float64), 2.0 ** -20, "uniform row")
    _check_route(torch.full((70, 12), float("-inf"), device=gpu, dtype=dtype), 3, True)     # nothing at all


def test_moe_route_nan_and_inf_stay_in_their_row(gpu):
    """A NaN or +inf logit shows in its row's weights and the losses; ids stay
    valid, other rows' weights and the plan are untouched."""
    import kernels
    x = _rand((200, 16), 3)
    want = kernels.moe_route(x, 4)
    for value in (float("nan"), float("inf")):
        y = x.clone()
        y[7, 5] = value
        r = kernels.moe_route(y, 4)
        assert int(r.ids[7, 0]) == 5 and int(r.ids.min()) >= 0 and int(r.ids.max()) < 16
        keep = torch.arange(200, device=gpu) != 7
        assert torch.equal(r.weights[keep], want.weights[keep]) and torch.equal(r.ids[keep], want.ids[keep])
        assert torch.isnan(r.weights[7]).any() and torch.isnan(r.balance_loss)
        _check_plan(r.plan, r.ids.cpu().numpy(), 16, 32)


def test_moe_route_strides_and_single_gradients(gpu):
    """Logits that are a view, and a backward pass through each output alone,
    with gradients that are expanded scalars."""
    import kernels
    wide = _rand((300, 50), 9, BF16)
    for view in (wide[:, 3:40], wide[::3, :37], _rand((37, 300), 10, BF16).t(), _rand((37,), 4, BF16).expand(5, 37)):
        _check_route(view, 4, True)
        r, c = kernels.moe_route(view, 4), kernels.moe_route(view.contiguous(), 4)
        assert torch.equal(r.weights, c.weights) and torch.equal(r.ids, c.ids)
    x = _rand((120, 20), 2).requires_grad_()
    for pick, gw, gb, gz in (("weights", torch.ones((120, 3), device=gpu), 0, 0), ("balance_loss", None, 1, 0),
                             ("z_loss", None, 0, 1)):
        x.grad = None
        getattr(kernels.moe_route(x, 3, normalize=False), pick).sum().backward()
        grad = _route_ref(x, 3, False, gw, gb, gz)[4]
        _close(x.grad, grad, 2.0 ** -24 * (grad.abs() + 200.0), pick)


def test_moe_route_gradient_against_differences(gpu):
    """Central differences of the 64-bit forward: L(l + h d) - L(l - h d) over 2h
    along random directions, within h^2 times a third derivative below 100."""
    import kernels
    x = _rand((6, 10), 1)
    gw = _rand((6, 3), 2)
    h = 1e-3
    for normalize in (True, False):
        def loss(l):
            w, ids, b, z, _ = _route_ref(l, 3, normalize)
            return float((w * gw.double()).sum() + 0.5 * b + 0.25 * z)

        y = x.clone().requires_grad_()
        r = kernels.moe_route(y, 3, normalize=normalize)
        ((r.weights * gw).sum() + 0.5 * r.balance_loss + 0.25 * r.z_loss).backward()
        for seed in range(8):
            d = _rand((6, 10), 50 + seed).double()
            # the choice must not change between the two points
            ids = [_route_ref(x.double() + s * h * d, 3, normalize)[1] for s in (-1, 1)]
            if not torch.equal(*ids):
                continue
            want = (loss(x.double() + h * d) - loss(x.double() - h * d)) / (2 * h)
            assert abs(float((y.grad.double() * d).sum()) - want) < 100 * h * h


# --- moving tokens ------------------------------------------------------------


def _some_plan(T, k, E, multiple, seed, dropped=True):
    """A plan of distinct experts per token, a few choices without an expert."""
    import kernels
    g = torch.Generator(device="cuda").manual_seed(seed)
    ids = torch.rand((T, E), generator=g, device="cuda").argsort(dim=1)[:, :k].to(torch.int32)
    if dropped and T > 2:
        ids[torch.rand((T, k), generator=g, device="cuda") < 0.1] = -1
        ids[1] = -1                             # a token that goes nowhere
    return kernels.token_plan(ids.contiguous(), E, multiple)


def _dispatch_ref(x, plan):
    k = plan.rows.shape[1]
    out = torch.zeros((plan.src.shape[0], x.shape[1]), dtype=torch.float64, device=x.device)
    valid = plan.src >= 0
    out[valid] = x.double()[(plan.src[valid] // k).long()]
    return out


def _gather_ref(y, plan, j):
    r = plan.rows[:, j].long()
    return torch.where((r >= 0).unsqueeze(1), y.double()[r.clamp_min(0)], 0.0)


@pytest.mark.parametrize("T,k,E,H,multiple,dtype", [
    (1, 1, 1, 1, 1, F32), (1, 2, 8, 512, 32, BF16), (2, 2, 2, 7, 32, F16), (33, 3, 5, 8, 32, BF16), (64, 2, 8, 4096, 32, BF16),
    (65, 8, 16, 513, 32, F32), (300, 1, 4, 520, 1, F16), (257, 5, 7, 2881, 32, BF16), (129, 4, 128, 1000, 32, F32),
    (1000, 8, 9, 264, 32, BF16), (40, 12, 12, 64, 32, F32),
])
def test_dispatch_and_combine(gpu, T, k, E, H, multiple, dtype):
    import kernels
    plan = _some_plan(T, k, E, multiple, seed=T + H)
    M = plan.src.shape[0]
    used = plan.src >= 0
    x = _rand((T, H), 1, dtype).requires_grad_()
    out = kernels.moe_dispatch(x, plan)
    assert torch.equal(out.detach().double(), _dispatch_ref(x.detach(), plan))
    g = _rand((M, H), 2, dtype)
    g[~used] = float("nan")                     # rows no token owns are not read
    out.backward(g)
    terms = [_gather_ref(g, plan, j) for j in range(k)]
    want, size = sum(terms), sum(t.abs() for t in terms)
    tol = HALF_ULP[dtype]
    _close(x.grad, want, tol * want.abs() * 1.01 + k * 2.0 ** -24 * size + TINY[dtype], "dispatch gradient")

    y = _rand((M, H), 3, dtype)
    y[~used] = float("nan")
    y.requires_grad_()
    w = _rand((T, k), 4)
    w[plan.rows < 0] = float("nan")             # gates of dropped choices are not read
    w.requires_grad_()
    o = kernels.moe_combine(y, w, plan)
    w0 = torch.where(plan.rows >= 0, w.detach(), 0.0).double()
    rows = [_gather_ref(y.detach(), plan, j) for j in range(k)]
    want = sum(w0[:, j:j + 1] * rows[j] for j in range(k))
    size = sum((w0[:, j:j + 1] * rows[j]).abs() for j in range(k))
    _close(o.detach(), want, tol * want.abs() * 1.01 + (k + 1) * 2.0 ** -24 * size + TINY[dtype], "combine")
    go = _rand((T, H), 5, dtype)
    o.backward(go)
    gy = _dispatch_ref(go, plan)
    gate = torch.zeros((M, 1), dtype=torch.float64, device=gpu)
    gate[used, 0] = w0.reshape(-1)[plan.src[used].long()]
    _close(y.grad, gy * gate, tol * (gy * gate).abs() * 1.01 + 2.0 ** -24 * (gy * gate).abs() + TINY[dtype], "grad of rows")
    assert not y.grad[~used].any()              # zeros, not what was there
    gw = torch.stack([(go.double() * rows[j]).sum(dim=1) for j in range(k)], dim=1)
    gs = torch.stack([(go.double() * rows[j]).abs().sum(dim=1) for j in range(k)], dim=1)
    _close(w.grad, gw, (H / 64 + 80) * 2.0 ** -24 * gs, "grad of gates")


def test_move_gradients_against_differences(gpu):
    """Both operators are linear in each argument, so a difference is exact up to
    the roundings of f32 sums of at most 64 terms below 8."""
    import kernels
    plan = _some_plan(20, 3, 6, 32, seed=8)
    M = plan.src.shape[0]
    x, d = _rand((20, 16), 1).requires_grad_(), _rand((20, 16), 2)
    c = _rand((M, 16), 3)
    (kernels.moe_dispatch(x, plan) * c).sum().backward()
    diff = ((kernels.moe_dispatch(x.detach() + d, plan) - kernels.moe_dispatch(x.detach(), plan)).double() * c.double()).sum()
    assert abs(float((x.grad.double() * d.double()).sum() - diff)) < 20 * 16 * 3 * 8 * 2.0 ** -22
    y, w = _rand((M, 16), 4).requires_grad_(), _rand((20, 3), 5).requires_grad_()
    dy, dw, c = _rand((M, 16), 6), _rand((20, 3), 7), _rand((20, 16), 8)
    (kernels.moe_combine(y, w, plan) * c).sum().backward()
    for grad, a, b in ((y.grad, (y.detach() + dy, w.detach()), dy), (w.grad, (y.detach(), w.detach() + dw), dw)):
        diff = ((kernels.moe_combine(*a, plan) - kernels.moe_combine(y.detach(), w.detach(), plan)).double() * c.double()).sum()
        assert abs(float((grad.double() * b.double()).sum() - diff)) < 20 * 16 * 3 * 32 * 2.0 ** -22


def test_move_strides(gpu):
    """Rows with a stride, on odd addresses, transposed, and expanded."""
    import kernels
    plan = _some_plan(90, 2, 4, 32, seed=3)
    M = plan.src.shape[0]
    wide, tall = _rand((95, 300), 1, BF16), _rand((M, 300), 2, BF16)
    w = _rand((2, 90), 3).t()
    for a, b in ((slice(0, 90), slice(0, 264)), (slice(5, 95), slice(1, 130)), (slice(0, 90), slice(7, 8))):
        x, y = wide[a, b], tall[:, b]
        assert torch.equal(kernels.moe_dispatch(x, plan), kernels.moe_dispatch(x.contiguous(), plan))
        assert torch.equal(kernels.moe_combine(y, w, plan), kernels.moe_combine(y.contiguous(), w.contiguous(), plan))
    t = _rand((130, 90), 4, F16).t()
    assert torch.equal(kernels.moe_dispatch(t, plan), kernels.moe_dispatch(t.contiguous(), plan))
    one = _rand((1, 64), 5, F32).expand(90, 64)
    assert torch.equal(kernels.moe_dispatch(one, plan), kernels.moe_dispatch(one.contiguous(), plan))
    x = _rand((90, 64), 6).requires_grad_()
    kernels.moe_dispatch(x, plan).sum().backward()                     # the gradient is an expanded scalar
    assert torch.equal(x.grad, (plan.rows >= 0).sum(dim=1, keepdim=True).float().expand(90, 64))


def test_move_past_32_bit_offsets(gpu):
    """More than 2^31 elements on the row side: rows at the end are found."""
    import kernels
    T, H = 66000, 33000
    ids = torch.zeros((T, 1), dtype=torch.int32, device=gpu)
    plan = kernels.token_plan(ids, 1, 32)
    x = torch.arange(T, device=gpu, dtype=torch.int32).to(torch.uint8).to(BF16).unsqueeze(1).expand(T, H).contiguous()
    y = kernels.moe_dispatch(x, plan)
    assert torch.equal(y[T - 40:T], x[T - 40:]) and torch.equal(y[:40], x[:40]) and not y[T:].any()
    o = kernels.moe_combine(y, torch.full((T, 1), 2.0, device=gpu), plan)
    assert torch.equal(o[T - 40:], 2 * x[T - 40:])


def test_streams_and_graph(gpu):
    """On a side stream, and captured: every replay on new inputs equals the eager result."""
    import kernels
    T, E, k, H = 64, 8, 2, 512
    logits, x = _rand((T, E), 1), _rand((T, H), 2, BF16)

    def step():
        r = kernels.moe_route(logits, k)
        rows = kernels.moe_dispatch(x, r.plan)
        return r.weights, r.plan.offs, r.balance_loss, kernels.moe_combine(rows * 2, r.weights, r.plan)

    want = [t.clone() for t in step()]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step()
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step()
    for seed in (3, 4, 5):
        logits.copy_(_rand((T, E), seed))
        x.copy_(_rand((T, H), seed + 10, BF16))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in static]
        assert all(torch.equal(a, b) for a, b in zip(step(), got))


def test_routing_refusals(gpu):
    import kernels
    x = _rand((16, 8), 1)
    plan = kernels.moe_route(x, 2).plan
    M = plan.src.shape[0]
    bad = [
        (ValueError, lambda: kernels.moe_route(x, 0)), (ValueError, lambda: kernels.moe_route(x, 9)),
        (ValueError, lambda: kernels.moe_route(x[0], 1)), (ValueError, lambda: kernels.moe_route(x, 2, multiple_of=0)),
        (TypeError, lambda: kernels.moe_route(x.double(), 2)), (TypeError, lambda: kernels.moe_route(x.cpu(), 2)),
        (ValueError, lambda: kernels.moe_route(_rand((4, 513), 1), 2)), (ValueError, lambda: kernels.moe_route(_rand((4, 64), 1), 33)),
        (TypeError, lambda: kernels.token_plan(x, 8)), (ValueError, lambda: kernels.token_plan(plan.rows.unsqueeze(0), 8)),
        (ValueError, lambda: kernels.token_plan(plan.rows, 0)), (ValueError, lambda: kernels.token_plan(plan.rows, 1025)),
        (ValueError, lambda: kernels.token_plan(plan.rows, 8, 0)), (TypeError, lambda: kernels.token_plan(plan.rows.cpu(), 8)),
        (ValueError, lambda: kernels.moe_dispatch(_rand((15, 8), 1), plan)), (TypeError, lambda: kernels.moe_dispatch(x.double(), plan)),
        (ValueError, lambda: kernels.moe_dispatch(x[0], plan)),
        (ValueError, lambda: kernels.moe_dispatch(x, kernels.TokenPlan(*(t.cpu() for t in plan)))),
        (TypeError, lambda: kernels.moe_dispatch(x, plan._replace(src=plan.src.long()))),
        (ValueError, lambda: kernels.moe_combine(_rand((M - 1, 8), 1), _rand((16, 2), 1), plan)),
        (ValueError, lambda: kernels.moe_combine(_rand((M, 8), 1), _rand((16, 3), 1), plan)),
        (TypeError, lambda: kernels.moe_combine(_rand((M, 8), 1), _rand((16, 2), 1, BF16), plan)),
    ]
    for i, (error, call) in enumerate(bad):
        with pytest.raises(error):
            call()
            pytest.fail(f"case {i} was accepted")
    x.requires_grad_()
    (g,) = torch.autograd.grad(kernels.moe_route(x, 2).z_loss, x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()                      # no second derivatives
