"""GPU checks of ``kernels.MXFP8MoE``: router, dispatch, MXFP8 experts, combine and
a shared projection with adapters, run together.

Against the same MXFP8 products made expert by expert (``mxfp8_grouped_mm`` on one
group: the same quantized operands, since every group starts on the 32-row grid)
with plain torch around them: gathers, softmax and sums in f32.  What may differ is
the order of f32 sums and so one step of a bf16 rounding: 2^-7 of a value for each
rounding on the way, of the sum of magnitudes where rounded terms are added up.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _block(E, k, hidden=256, inter=192):
    import kernels
    torch.manual_seed(0)
    return kernels.MXFP8MoE(hidden, inter, E, k, device="cuda")


def _adapters(T, L, hidden, seed=1):
    import kernels
    g = torch.Generator(device="cuda").manual_seed(seed)
    ids = torch.randint(-1, L, (T,), generator=g, device="cuda")
    down = (torch.randn((L, 8, hidden), generator=g, device="cuda") * hidden ** -0.5).to(BF16)
    up = (torch.randn((L, 8, hidden), generator=g, device="cuda") * 0.3).to(BF16)
    return ids, kernels.Adapters(down, up, kernels.token_plan(ids, L), torch.linspace(0.5, 1.5, L, device="cuda"))


def _pad32(x):
    return torch.nn.functional.pad(x, (0, 0, 0, -x.shape[0] % 32))


def _product(x, w):
    """x (n, K) in f32 times w[0]^T in MXFP8, in f32."""
    import kernels
    p = _pad32(x.to(BF16))
    offs = torch.full((1,), p.shape[0], dtype=torch.int32, device=x.device)
    return kernels.mxfp8_grouped_mm(p, w, offs)[:x.shape[0]].float()


def _by_experts(block, routing, ids, ad, p):
    """(y, base) from f32 leaves p, expert by expert; the choice is given."""
    logits = (p["x"].to(BF16) @ p["gate"].to(BF16).t()).float()
    w = torch.softmax(logits, dim=1).gather(1, routing.ids.long())
    w = w / w.sum(dim=1, keepdim=True)
    y = torch.zeros_like(p["x"])
    for e in range(p["w_in"].shape[0]):
        t, j = torch.nonzero(routing.ids == e, as_tuple=True)
        if t.numel():
            a, b = _product(p["x"][t], p["w_in"][e:e + 1].to(BF16)).to(BF16).chunk(2, dim=1)
            h = _product((torch.nn.functional.silu(a) * b).float(), p["w_out"][e:e + 1].to(BF16))
            y = y.index_add(0, t, w[t, j].unsqueeze(1) * h)
    base = _product(p["x"], p["shared"].to(BF16))
    for a in range(ad.down.shape[0]):
        t = torch.nonzero(ids == a)[:, 0]
        base = base.index_add(0, t, ad.scales[a] * (p["x"][t] @ p["down"][a].t()) @ p["up"][a])
    return y, base


@pytest.mark.parametrize("T,E,k", [(1, 4, 2), (100, 8, 2), (513, 4, 3)])
def test_moe_block_forward_and_gradients(gpu, T, E, k):
    block = _block(E, k)
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn((T, 256), generator=g, device="cuda").to(BF16).requires_grad_()
    ids, ad = _adapters(T, 3, 256)
    ad = ad._replace(down=ad.down.requires_grad_(), up=ad.up.requires_grad_())
    go = torch.randn((T, 256), generator=g, device="cuda").to(BF16)
    out, routing = block(x, ad)
    out.backward(go)
    p = {"x": x, "gate": block.gate.weight, "w_in": block.w_in.weight, "w_out": block.w_out.weight,
         "shared": block.shared.weight, "down": ad.down, "up": ad.up}
    ref = {n: t.detach().float().requires_grad_() for n, t in p.items()}
    y, base = _by_experts(block, routing, ids, ad, ref)
    want = y + base
    step = 2.0 ** -7
    bad = (out.detach().float() - want.detach()).abs() > step * (y.abs() + base.abs() + want.abs()) + 1e-6
    assert not bad.any(), int(bad.sum())
    want.backward(go.float())
    for n, t in p.items():
        # a gradient of x adds up k + 3 rounded terms, one of the gate T of them
        size = ref[n].grad.abs() + ref[n].grad.abs().mean() * (k + 3)
        bad = (t.grad.float() - ref[n].grad).abs() > 4 * step * size
        assert torch.isfinite(t.grad).all() and not bad.any(), (n, int(bad.sum()), t.numel())


def test_moe_block_padding_tokens(gpu):
    """Masked tokens get the shared projection only, and do not change the others."""
    block = _block(8, 2)
    x = torch.randn((70, 256), device=gpu, generator=torch.Generator("cuda").manual_seed(3)).to(BF16)
    mask = torch.arange(70, device=gpu) < 50
    with torch.no_grad():
        y, routing = block(x, mask=mask)
        full, _ = block(x)
        base = full.clone()
        block.gate.weight.zero_()
        none, r = block(x, mask=torch.zeros(70, dtype=torch.bool, device=gpu))
    assert (routing.ids[50:] == -1).all() and int(routing.plan.counts.sum()) == 100
    assert torch.equal(y[:50], base[:50]) and torch.equal(y[50:], none[50:])
    assert int(r.plan.offs[-1]) == 0 and float(r.balance_loss) == 0.0 and torch.isfinite(none).all()


def test_moe_block_trains(gpu):
    """Steps on the task's loss lower it, and steps on the balance loss even out a
    router that prefers one expert."""
    x = torch.randn((512, 256), device=gpu, generator=torch.Generator("cuda").manual_seed(4)).abs().to(BF16)
    target = torch.randn((512, 256), device=gpu, generator=torch.Generator("cuda").manual_seed(5))
    block = _block(8, 2)
    opt = torch.optim.SGD(block.parameters(), lr=0.3)
    seen = []
    for _ in range(8):
        opt.zero_grad()
        y, r = block(x)
        task = ((y.float() - target) ** 2).mean()
        (task + 0.01 * r.balance_loss + 1e-3 * r.z_loss).backward()
        opt.step()
        seen.append(float(task))
    assert seen[-1] < seen[0], seen
    block = _block(8, 2)
    with torch.no_grad():
        block.gate.weight[0] += 0.01            # a lead of about 2 over the other logits
    opt = torch.optim.SGD([block.gate.weight], lr=0.02)
    seen = []
    for _ in range(8):
        opt.zero_grad()
        r = block(x)[1]
        r.balance_loss.backward()
        opt.step()
        seen.append(float(r.balance_loss))
    assert seen[-1] < seen[0], seen
