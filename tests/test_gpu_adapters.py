"""GPU checks of ``kernels.lora_grouped_mm``: the adapters of a batch and their
gradients against the formulas in 64 bits.

Bounds per element, from the formulas on absolute values: a chain of f32 sums
over n terms errs by n 2^-24 of the sum of magnitudes, the hidden row enters the
second product to 2^-16 (two 8-bit terms; f16: relative to its row's largest
value), and the result is rounded once to its type.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
HALF_ULP = {BF16: 2.0 ** -8, F16: 2.0 ** -11}      # relative, 8 / 11 bits
TINY = {BF16: 2.0 ** -134, F16: 2.0 ** -25}


def _rand(shape, seed, dtype, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def _ids(T, L, seed, kind):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if kind == "mixed":
        return torch.randint(-1, L, (T,), generator=g, device="cuda", dtype=torch.int32)
    if kind == "none":
        return torch.full((T,), -1, dtype=torch.int32, device="cuda")
    if kind == "one":
        return torch.full((T,), L - 1, dtype=torch.int32, device="cuda")
    return torch.sort(torch.randint(-1, L, (T,), generator=g, device="cuda", dtype=torch.int32)).values   # runs


def _inputs(T, L, r, K, N, dtype, seed):
    return {"x": _rand((T, K), seed, dtype), "down": _rand((L, r, K), seed + 1, dtype, K ** -0.5),
            "up": _rand((L, r, N), seed + 2, dtype, 0.2), "base": _rand((T, N), seed + 3, dtype),
            "scales": torch.linspace(0.5, 2.0, L, device="cuda")}


def _reference(s, ids, g=None):
    """(values, sums of magnitudes) of out and, with g, of gx, gdown, gup."""
    x, down, up, sc = s["x"].double(), s["down"].double(), s["up"].double(), s["scales"].double()
    N = up.shape[2]
    out = s["base"].double().clone() if s.get("base") is not None else x.new_zeros((x.shape[0], N))
    val, mag = {"out": out}, {"out": out.abs()}
    if g is not None:
        g = g.double()
        for name, like in (("x", x), ("down", down), ("up", up)):
            val[name], mag[name] = torch.zeros_like(like), torch.zeros_like(like)
    for a in range(down.shape[0]):
        t = torch.nonzero(ids == a)[:, 0]
        if not t.numel():
            continue
        for d, f in ((val, lambda v: v), (mag, torch.abs)):
            X, D, U, S = f(x[t]), f(down[a]), f(up[a]), sc[a].abs()
            h = X @ D.t()
            d["out"][t] += S * (h @ U)
            if g is not None:
                G = f(g[t])
                u = G @ U.t()
                d["x"][t] += S * (u @ D)
                d["down"][a] += S * (u.t() @ X)
                d["up"][a] += S * (h.t() @ G)
    return val, mag


def _close(got, want, mag, n, what):
    dt = got.dtype
    bound = HALF_ULP[dt] * want.abs() * 1.01 + (n * 2.0 ** -24 + 2.0 ** -15) * mag + TINY[dt]
    bad = ~((got.double() - want).abs() <= bound)
    assert not bad.any(), (what, int(bad.sum()), float((got.double() - want).abs().max()))


def _check(T, L, r, K, N, dtype, kind="mixed", seed=0, with_base=True, grads=True):
    import kernels
    s = _inputs(T, L, r, K, N, dtype, seed)
    if not with_base:
        s["base"] = None
    ids = _ids(T, L, seed, kind)
    plan = kernels.token_plan(ids, L)
    leaves = {n: s[n].clone().requires_grad_(grads) for n in ("x", "down", "up")}
    base = s["base"].clone().requires_grad_(grads) if with_base else None
    out = kernels.lora_grouped_mm(leaves["x"], leaves["down"], leaves["up"], plan, scales=s["scales"], base=base)
    g = _rand((T, N), seed + 9, dtype)
    val, mag = _reference(s, ids, g if grads else None)
    _close(out.detach(), val["out"], mag["out"], K + r + 16, "out")
    if not grads:
        return
    out.backward(g)
    n = {"x": N + r + 16, "down": N + T + 16, "up": K + T + 16}
    for name, t in leaves.items():
        _close(t.grad, val[name], mag[name], n[name], name)
    if with_base:
        assert torch.equal(base.grad, g)


@pytest.mark.parametrize("T,L,r,K,N,dtype,kind", [
    (1, 1, 1, 1, 1, BF16, "one"), (1, 4, 16, 512, 640, BF16, "one"), (1, 3, 8, 64, 64, F16, "none"), (15, 2, 8, 64, 128, BF16, "mixed"),
    (16, 1, 16, 65, 63, F16, "one"), (17, 3, 17, 200, 520, BF16, "mixed"), (64, 70, 16, 1024, 1000, BF16, "mixed"),
    (65, 2, 33, 129, 257, F16, "runs"), (300, 3, 64, 513, 2881, BF16, "runs"), (257, 5, 20, 2880, 515, F16, "mixed"),
    (130, 2, 100, 264, 136, BF16, "runs"), (200, 1, 128, 256, 512, F16, "one"), (96, 2, 200, 192, 200, BF16, "runs"),
    (70, 2, 512, 72, 96, F16, "mixed"), (70, 2, 300, 72, 96, BF16, "mixed"), (700, 4, 32, 320, 384, BF16, "runs"),
    (1500, 3, 16, 1160, 2056, BF16, "runs"), (1500, 200, 8, 136, 264, F16, "mixed"), (900, 1, 16, 5120, 128, BF16, "one"),
    (2500, 2, 48, 256, 8192, F16, "runs"),
])
def test_lora_grouped_mm(gpu, T, L, r, K, N, dtype, kind):
    _check(T, L, r, K, N, dtype, kind, seed=T + r)


def test_lora_without_base_or_scales(gpu):
    import kernels
    _check(100, 3, 16, 256, 384, BF16, with_base=False)
    _check(100, 3, 16, 256, 384, F16, "none", with_base=False)
    s = _inputs(50, 3, 8, 64, 128, BF16, 1)
    plan = kernels.token_plan(_ids(50, 3, 1, "mixed"), 3)
    one = kernels.lora_grouped_mm(s["x"], s["down"], s["up"], plan, base=s["base"])
    ones = kernels.lora_grouped_mm(s["x"], s["down"], s["up"], plan, scales=torch.ones(3, device=gpu), base=s["base"])
    assert torch.equal(one, ones)


def test_lora_in_place_and_out(gpu):
    """out= takes the result; base itself adds in place, and rows without an
    adapter keep their bits."""
    import kernels
    for T, dtype in ((37, BF16), (700, F16)):
        s = _inputs(T, 3, 16, 192, 520, dtype, 2)
        ids = _ids(T, 3, 2, "mixed")
        plan = kernels.token_plan(ids, 3)
        args = (s["x"], s["down"], s["up"], plan)
        want = kernels.lora_grouped_mm(*args, scales=s["scales"], base=s["base"])
        wide = torch.full((T, 600), 7.0, dtype=dtype, device=gpu)
        got = kernels.lora_grouped_mm(*args, scales=s["scales"], base=s["base"], out=wide[:, :520])
        assert torch.equal(got, want) and (wide[:, 520:] == 7.0).all()
        buf = s["base"].clone()
        assert kernels.lora_grouped_mm(*args, scales=s["scales"], base=buf, out=buf) is buf
        assert torch.equal(buf, want) and torch.equal(buf[ids < 0], s["base"][ids < 0])


def test_lora_padded_plan(gpu):
    """A plan whose groups are padded serves as well."""
    import kernels
    s = _inputs(90, 4, 16, 128, 256, BF16, 3)
    ids = _ids(90, 4, 3, "mixed")
    val, mag = _reference(dict(s, scales=torch.ones(4, device=gpu)), ids)
    for m in (1, 32):
        out = kernels.lora_grouped_mm(s["x"], s["down"], s["up"], kernels.token_plan(ids, 4, m), base=s["base"])
        _close(out, val["out"], mag["out"], 160, "padded")
    x = s["x"].clone().requires_grad_()
    d, u = s["down"].clone().requires_grad_(), s["up"].clone().requires_grad_()
    g = _rand((90, 256), 5, BF16)
    kernels.lora_grouped_mm(x, d, u, kernels.token_plan(ids, 4, 32)).backward(g)
    val, mag = _reference(dict(s, base=None, scales=torch.ones(4, device=gpu)), ids, g)
    for name, t, n in (("x", x, 300), ("down", d, 400), ("up", u, 300)):
        _close(t.grad, val[name], mag[name], n, name)


def test_lora_strides(gpu):
    """Column slices on odd addresses, transposed factors, expanded adapters and
    gradients."""
    import kernels
    s = _inputs(70, 3, 16, 300, 300, BF16, 4)
    plan = kernels.token_plan(_ids(70, 3, 4, "mixed"), 3)
    x, base = s["x"][:, 5:205], s["base"][:, 1:131]
    for down, up in ((s["down"][:, :, 3:203], s["up"][:, :, 7:137]), (s["down"][:, ::2, 3:203], s["up"][:, 1::2, 7:137]),
                     (_rand((3, 200, 16), 5, BF16).transpose(1, 2), _rand((3, 130, 16), 6, BF16).transpose(1, 2)),
                     (s["down"][:1, :, :200].expand(3, 16, 200), s["up"][:1, :1, :130].expand(3, 16, 130))):
        a = kernels.lora_grouped_mm(x, down, up, plan, base=base)
        b = kernels.lora_grouped_mm(x.contiguous(), down.contiguous(), up.contiguous(), plan, base=base.contiguous())
        assert torch.equal(a, b)
    leaf = s["x"].clone().requires_grad_()
    kernels.lora_grouped_mm(leaf, s["down"], s["up"], plan).float().sum().backward()
    ref = s["x"].clone().requires_grad_()
    kernels.lora_grouped_mm(ref, s["down"], s["up"], plan).backward(torch.ones((70, 300), dtype=BF16, device=gpu))
    assert torch.equal(leaf.grad, ref.grad)


def test_lora_special_values_stay_where_they_are(gpu):
    """NaN in one token or one adapter reaches that token or adapter only; an
    infinity gives what the formula gives; adapters no token uses are not read."""
    import kernels
    s = _inputs(80, 4, 20, 136, 264, BF16, 5)
    ids = _ids(80, 3, 5, "mixed")               # adapter 3 is not used
    plan = kernels.token_plan(ids, 4)
    want = kernels.lora_grouped_mm(s["x"], s["down"], s["up"], plan, base=s["base"])
    x, down, up = s["x"].clone(), s["down"].clone(), s["up"].clone()
    row = int(torch.nonzero(ids == 0)[0])
    x[row, 11] = float("nan")
    none = int(torch.nonzero(ids < 0)[0])
    x[none] = float("nan")                      # a token without an adapter
    down[3] = float("nan")
    up[3] = float("nan")
    down[1, 2] = float("nan")
    got = kernels.lora_grouped_mm(x, down, up, plan, base=s["base"])
    hit = (ids == 1) | (torch.arange(80, device=gpu) == row)
    assert torch.isnan(got[hit]).all() and torch.equal(got[~hit], want[~hit])
    x = s["x"].clone()
    x[row, 11] = float("inf")
    up = s["up"].abs()                          # infinite hidden values of both signs, no cancelling zeros
    got = kernels.lora_grouped_mm(x, s["down"].abs(), up, plan, base=s["base"])
    assert torch.isinf(got[row]).all() and torch.isfinite(got[torch.arange(80, device=gpu) != row]).all()


def test_lora_f16_hidden_values_beyond_the_type(gpu):
    """Hidden values above 65504 and below the smallest f16 do not overflow or
    vanish on the way to the output."""
    import kernels
    for big, small in ((400.0, 2.0 ** -12), (2.0 ** -10, 256.0)):
        x = torch.full((20, 2048), big, dtype=F16, device=gpu) * torch.linspace(0.5, 1, 20, device=gpu).to(F16).unsqueeze(1)
        down = torch.full((1, 8, 2048), 0.5 if big > 1 else 2.0 ** -18, dtype=F16, device=gpu)
        up = torch.full((1, 8, 96), small, dtype=F16, device=gpu)
        s = {"x": x, "down": down, "up": up, "base": None, "scales": torch.ones(1, device=gpu)}
        ids = torch.zeros(20, dtype=torch.int32, device=gpu)
        val, mag = _reference(s, ids)
        assert float((x.double() @ down[0].double().t()).abs().max()) > 65504 or big < 1
        _close(kernels.lora_grouped_mm(x, down, up, kernels.token_plan(ids, 1)), val["out"], mag["out"], 2100, "out")


def test_lora_gradient_against_differences(gpu):
    """Along a random direction of each argument the formula is linear: the
    64-bit difference equals the product with the gradient, within the
    gradient's rounding to bf16."""
    import kernels
    s = _inputs(40, 2, 8, 64, 96, BF16, 6)
    ids = _ids(40, 2, 6, "mixed")
    plan = kernels.token_plan(ids, 2)
    g = _rand((40, 96), 7, BF16)
    leaves = {n: s[n].clone().requires_grad_() for n in ("x", "down", "up")}
    kernels.lora_grouped_mm(*leaves.values(), plan, scales=s["scales"], base=s["base"]).backward(g)
    for name, leaf in leaves.items():
        d = _rand(leaf.shape, 8, BF16).double()
        moved = dict(s)
        moved[name] = s[name].double() + d
        diff = ((_reference(moved, ids)[0]["out"] - _reference(s, ids)[0]["out"]) * g.double()).sum()
        size = (leaf.grad.double().abs() * d.abs()).sum()
        assert abs(float((leaf.grad.double() * d).sum() - diff)) < 2.0 ** -8 * float(size)


def test_lora_is_repeatable_on_any_stream_and_in_graphs(gpu):
    import kernels
    s = _inputs(600, 3, 16, 512, 768, BF16, 7)
    ids = _ids(600, 3, 7, "mixed")
    g = _rand((600, 768), 8, BF16)

    def step():
        leaves = [s[n].clone().requires_grad_() for n in ("x", "down", "up")]
        out = kernels.lora_grouped_mm(*leaves, kernels.token_plan(ids, 3), scales=s["scales"], base=s["base"])
        out.backward(g)
        return [out.detach()] + [t.grad for t in leaves]

    want = step()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(want, step()))
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = step()
    st.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))

    def serve():
        return kernels.lora_grouped_mm(s["x"], s["down"], s["up"], kernels.token_plan(ids, 3), scales=s["scales"], base=s["base"])

    serve()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = serve()
    for seed in (1, 2, 3):
        ids.copy_(_ids(600, 3, seed, "mixed"))
        s["x"].copy_(_rand((600, 512), seed, BF16))
        graph.replay()
        torch.cuda.synchronize()
        got = static.clone()
        assert torch.equal(got, serve())


def test_lora_past_32_bit_offsets(gpu):
    """More than 2^31 output elements: the last tokens' rows are right."""
    import kernels
    T, N = 70000, 32768
    x = _rand((T, 64), 1, BF16)
    down, up = _rand((2, 4, 64), 2, BF16, 0.125), _rand((2, 4, N), 3, BF16, 0.2)
    ids = torch.arange(T, device=gpu, dtype=torch.int32) % 2
    plan = kernels.token_plan(ids, 2)
    out = torch.ones((T, N), dtype=BF16, device=gpu)
    kernels.lora_grouped_mm(x, down, up, plan, base=out, out=out)
    for rows in (slice(0, 20), slice(T - 20, T)):
        s = {"x": x[rows], "down": down, "up": up, "base": torch.ones((20, N), dtype=BF16, device=gpu),
             "scales": torch.ones(2, device=gpu)}
        val, mag = _reference(s, ids[rows])
        _close(out[rows], val["out"], mag["out"], 100, "rows")


@pytest.mark.parametrize("tail", range(1, 8))
def test_lora_row_ends(gpu, tail):
    """Rows that end inside a 16-byte piece, many and few tokens an adapter, and
    rows shorter than a piece."""
    dtype = F16 if tail % 2 else BF16
    _check(90, 2, 20, 128 + tail, 256 - tail, dtype, "runs", seed=tail)
    _check(12, 6, 40, 64 - tail, 512 + tail, dtype, seed=tail)
    _check(70, 2, 70, tail, 9 - tail, dtype, "runs", seed=tail)
    _check(9, 4, 5, 8 - tail, tail, dtype, seed=tail)


@pytest.mark.parametrize("T,L,r,K,N,dtype", [
    (1, 1, 65, 3976, 1032, F16), (9, 8, 130, 5000, 520, BF16), (40, 40, 256, 1544, 264, F16), (33, 33, 64, 4104, 1000, BF16),
    (2300, 17, 99, 1032, 392, F16), (1000, 3, 257, 640, 648, BF16),
])
def test_lora_high_ranks(gpu, T, L, r, K, N, dtype):
    _check(T, L, r, K, N, dtype, seed=T)


@pytest.mark.parametrize("N", [8184, 8191, 8192])
def test_lora_outputs_beyond_the_caches(gpu, N):
    _check(2500, 3, 8, 64, N, BF16, "runs", grads=False)


@pytest.mark.parametrize("counts", [(0, 1, 3000, 30, 0, 700, 256, 257), (2000, 0), (0, 0, 5), (300, 300, 300)])
def test_lora_uneven_adapters(gpu, counts):
    """Adapters of no token, of one chunk and of many: every gradient is whole."""
    import kernels
    L, r, K, N = len(counts), 40, 264, 520
    ids = torch.cat([torch.full((c,), a, dtype=torch.int32, device=gpu) for a, c in enumerate(counts)])
    ids = ids[torch.randperm(len(ids), generator=torch.Generator().manual_seed(1)).to(gpu)]
    T = len(ids)
    s = _inputs(T, L, r, K, N, BF16, 11)
    leaves = {n: s[n].clone().requires_grad_() for n in ("x", "down", "up")}
    g = _rand((T, N), 12, BF16)
    out = kernels.lora_grouped_mm(*leaves.values(), kernels.token_plan(ids, L), scales=s["scales"], base=s["base"])
    out.backward(g)
    val, mag = _reference(s, ids, g)
    n = {"x": N + r + 16, "down": N + T + 16, "up": K + T + 16}
    for name, t in leaves.items():
        _close(t.grad, val[name], mag[name], n[name], name)
    for a, c in enumerate(counts):
        if c == 0:
            assert not leaves["down"].grad[a].any() and not leaves["up"].grad[a].any()


def test_lora_refusals(gpu):
    import kernels
    s = _inputs(20, 3, 8, 64, 96, BF16, 8)
    plan = kernels.token_plan(_ids(20, 3, 8, "mixed"), 3)
    x, down, up, base = s["x"], s["down"], s["up"], s["base"]
    call = kernels.lora_grouped_mm
    two = kernels.token_plan(torch.zeros((20, 2), dtype=torch.int32, device=gpu), 3)
    bad = [
        (TypeError, lambda: call(x.float(), down, up, plan)), (TypeError, lambda: call(x.cpu(), down, up, plan)),
        (TypeError, lambda: call(x, down.half(), up, plan)), (TypeError, lambda: call(x, down, up.half(), plan)),
        (TypeError, lambda: call(x, down, up, plan, base=base.half())), (ValueError, lambda: call(x[:19], down, up, plan)),
        (ValueError, lambda: call(x[:, :63], down, up, plan)), (ValueError, lambda: call(x, down[:, :7], up, plan)),
        (ValueError, lambda: call(x, down[:2], up[:2], plan)), (ValueError, lambda: call(x, down[0], up[0], plan)),
        (ValueError, lambda: call(x, down, up, two)), (ValueError, lambda: call(x, down, up, plan, base=base[:, :95])),
        (ValueError, lambda: call(x, down, up, plan, scales=torch.ones(2, device=gpu))),
        (ValueError, lambda: call(x, down, up, plan, scales=torch.ones(3, device=gpu).double())),
        (ValueError, lambda: call(x, down.cpu(), up, plan)),
        (ValueError, lambda: call(x, down, up, plan, out=torch.empty((96, 20), dtype=BF16, device=gpu).t())),
        (ValueError, lambda: call(x.clone().requires_grad_(), down, up, plan, out=base)),
        (ValueError, lambda: call(_rand((20, 64), 1, BF16), _rand((3, 513, 64), 1, BF16), _rand((3, 513, 8), 1, BF16), plan)),
    ]
    for i, (error, f) in enumerate(bad):
        with pytest.raises(error):
            f()
            pytest.fail(f"case {i} was accepted")
    empty = kernels.token_plan(torch.zeros((0,), dtype=torch.int32, device=gpu), 3)
    assert tuple(call(x[:0], down, up, empty, base=base[:0]).shape) == (0, 96)
    leaves = [x[:0].clone().requires_grad_(), down.clone().requires_grad_(), up.clone().requires_grad_()]
    call(*leaves, empty, base=base[:0]).sum().backward()       # no tokens: zero gradients
    assert not leaves[1].grad.any() and not leaves[2].grad.any() and leaves[0].grad.shape == (0, 64)
