"""The operators around the grouped GEMMs, as cases that can be timed and checked.

* ``moe_route``: a router's logits to gate weights, expert ids, the token plan
  (rows sorted by expert), per-expert counts, the balance and z losses; with
  the gradient of the logits.
* ``moe_dispatch`` / ``moe_combine``: tokens to expert rows and back, weighted;
  with their gradients.
* ``lora_grouped_mm``: the low-rank adapters of many requests beside a shared
  projection; with the gradients of the input and of the adapters.

``own`` chooses what ``run`` times: the plain torch form of each operator in
32 bits, or the package's entry points.  Run with the repository's root as the
working directory.
"""

import math
import os
import random
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}
_MULTIPLE = 32      # expert groups start on the 32-row grid of the MX scale blocks


def _kernels():
    pkg = os.path.join(os.getcwd(), "grouped-gemms_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import kernels
    return kernels


# --- cases ------------------------------------------------------------------


def listed():
    """The fixed cases, from one token to whole training batches."""
    return [
        # Serving one sequence: the router of one token, launches and host time.
        _route("route one token", 1, 32, 4, "bf16", "fwd"),
        # Training with few large experts, the benchmark's batch; f32 logits.
        _route("route training", 16640, 8, 2, "f32", "step"),
        # Training with many small experts.
        _route("route many experts", 16640, 256, 8, "bf16", "step"),
        # A padded batch: sizes that fill nothing, padding rows whose logits
        # are all masked, experts masked for some tokens, gates that are not
        # renormalised.
        _route("route masked", 4099, 37, 5, "f16", "step", normalize=False, masked=True),
        # One decode step of a serving batch.
        _move("dispatch decode", "dispatch", 64, 8, 2, 8192, "bf16", "fwd"),
        # A training batch to its experts, and the gradient back.
        _move("dispatch training", "dispatch", 16640, 8, 2, 5120, "bf16", "step"),
        # The way back of a decode step.
        _move("combine decode", "combine", 64, 8, 2, 8192, "bf16", "fwd"),
        # The way back of a training batch over many experts, with the
        # gradients of the rows and of the gates.
        _move("combine training", "combine", 8320, 32, 8, 2048, "bf16", "step"),
        # A decode batch whose requests use 64 adapters of rank 16, some none.
        _lora("adapters decode", 64, 64, 16, 8192, 8192, "bf16", "fwd", "tokens"),
        # Prompts of many requests at once, adapters of rank 64.
        _lora("adapters prefill", 16640, 8, 64, 5120, 8192, "bf16", "fwd", "requests"),
        # Training four adapters beside a frozen projection.
        _lora("adapters training", 8320, 4, 16, 2048, 8192, "bf16", "step", "requests"),
        # Ragged serving batch: a rank off the matrix unit's grid, short
        # requests, a hidden size that fills no tile; f16 model.
        _lora("adapters ragged", 997, 33, 20, 2880, 2880, "f16", "fwd", "requests"),
    ]


def _named(name, c):
    return dict(c, name=name) if name else c


def _route(name, T, E, k, dtype, mode, normalize=True, masked=False):
    return _named(name, {"op": "route", "T": T, "E": E, "k": k, "dtype": dtype, "mode": mode, "normalize": normalize,
                         "masked": masked})


def _move(name, op, T, E, k, H, dtype, mode):
    return _named(name, {"op": op, "T": T, "E": E, "k": k, "H": H, "dtype": dtype, "mode": mode})


def _lora(name, T, L, r, K, N, dtype, mode, batch):
    """batch: "tokens", every token a request of its own (decode); "requests",
    runs of tokens with one adapter each (prompts, training)."""
    return _named(name, {"op": "lora", "T": T, "L": L, "r": r, "K": K, "N": N, "dtype": dtype, "mode": mode,
                         "batch": batch})


def _log(rng, lo, hi, step=1):
    """An integer of [lo, hi], spread over its logarithm, a multiple of step."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(-(-lo // step), min(hi // step, round(v / step))) * step


def draw(rng):
    """One more case: any operator over the listed cases' ranges."""
    op = rng.choice(("route", "route", "dispatch", "combine", "lora", "lora", "lora"))
    if op == "route":
        E = _log(rng, 2, 256)
        return _route(None, _log(rng, 1, 16640), E, rng.randint(1, min(E, 8)), rng.choice(("bf16", "f16", "f32")),
                      rng.choice(("fwd", "step", "step")), rng.random() < 0.7, rng.random() < 0.3)
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    if op != "lora":
        E = rng.choice((1, 2, 4, 8, 16, 32, 128))
        k = rng.randint(1, min(E, 8))
        H = _log(rng, 512, 8192, rng.choice((8, 8, 1)))
        # at most the rows and columns of the largest listed batch
        T = _log(rng, 1, max(1, min(16640, 16640 * 2 * 5120 // (2 * k * H * (_BYTES[dtype] // 2)))))
        return _move(None, op, T, E, k, H, dtype, rng.choice(("fwd", "step")))
    dtype = "bf16" if dtype == "f32" else dtype
    step = rng.choice((32, 8, 8, 1))
    K, N, r = _log(rng, 512, 8192, step), _log(rng, 512, 8192, step), _log(rng, 4, 128)
    L = _log(rng, 1, 64)
    if rng.random() < 0.4:
        return _lora(None, _log(rng, 1, 256), L, r, K, N, dtype, "fwd", "tokens")
    mode = rng.choice(("fwd", "fwd", "step"))
    top = 16640 * 64 * (5120 + 8192) // (r * (K + N) * (3 if mode == "step" else 1))
    return _lora(None, _log(rng, 128, max(128, min(8320 if mode == "step" else 16640, top))), L, r, K, N, dtype, mode,
                 "requests")


# --- inputs -----------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(shape, std, gen, dtype):
    return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * std).to(dtype)


def _capacity(entries, groups, multiple):
    """Rows of a plan: the entries, and each used group rounded up."""
    return (entries + min(groups, entries) * (multiple - 1)) // multiple * multiple


def _logits(case, gen):
    """Logits of a router that prefers some experts; where masked, one expert
    in eight is closed to a token and the batch's last eighth is padding."""
    T, E = case["T"], case["E"]
    x = torch.randn((T, E), generator=gen, device="cuda") * 1.5
    x += torch.randn((1, E), generator=gen, device="cuda") * 0.7
    if case["masked"]:
        x[torch.rand((T, E), generator=gen, device="cuda") < 0.125] = float("-inf")
        x[T - T // 8:] = float("-inf")
    return x.to(_DTYPES[case["dtype"]])


def _choices(case, gen):
    """Expert ids (T, k), every token's experts different, some experts popular."""
    x = torch.randn((case["T"], case["E"]), generator=gen, device="cuda")
    x += torch.randn((1, case["E"]), generator=gen, device="cuda") * 0.7
    return x.argsort(dim=1, descending=True)[:, :case["k"]].to(torch.int32).contiguous()


def _adapters(case, seed):
    """Adapter of every token as a list, -1 for none."""
    rnd = random.Random(seed)
    T, L = case["T"], case["L"]

    def one():
        return -1 if rnd.random() < 0.125 else rnd.randrange(L)

    if case["batch"] == "tokens":
        return [one() for _ in range(T)]
    ids = []
    while len(ids) < T:
        ids += [one()] * min(T - len(ids), 1 + int(rnd.expovariate(L / (2.0 * T))))
    return ids


def _inputs(case, seed):
    """The tensors of a case, from its seed alone."""
    gen, dt = _gen(seed), _DTYPES[case["dtype"]]
    s = {}
    if case["op"] == "route":
        s["logits"] = _logits(case, gen)
        if case["mode"] == "step":
            s["g_weights"] = torch.randn((case["T"], case["k"]), generator=gen, device="cuda") / case["T"]
            # the losses' coefficients in the training objective
            s["g_balance"] = torch.tensor(0.01, device="cuda")
            s["g_z"] = torch.tensor(0.001, device="cuda")
        return s
    T = case["T"]
    if case["op"] == "lora":
        L, r, K, N = case["L"], case["r"], case["K"], case["N"]
        s["x"] = _randn((T, K), 1.0, gen, dt)
        s["base"] = _randn((T, N), 1.0, gen, dt)
        s["down"] = _randn((L, r, K), K ** -0.5, gen, dt)
        s["up"] = _randn((L, r, N), 0.1, gen, dt)
        s["scales"] = torch.rand((L,), generator=gen, device="cuda") * 1.5 + 0.5
        s["adapter"] = _adapters(case, seed)
        if case["mode"] == "step":
            s["g"] = _randn((T, N), 1.0, gen, dt)
        return s
    s["ids"] = _choices(case, gen)
    rows = _capacity(T * case["k"], case["E"], _MULTIPLE)
    if case["op"] == "dispatch":
        s["x"] = _randn((T, case["H"]), 1.0, gen, dt)
        if case["mode"] == "step":
            s["g"] = _randn((rows, case["H"]), 1.0, gen, dt)
        return s
    s["y"] = _randn((rows, case["H"]), 1.0, gen, dt)
    s["weights"] = torch.randn((T, case["k"]), generator=gen, device="cuda").softmax(dim=1)
    if case["mode"] == "step":
        s["g"] = _randn((T, case["H"]), 1.0, gen, dt)
    return s


def prepare(case, seed):
    """What a program holds before the call: the tensors; for moving tokens and
    for the adapters also the token plan, made once for all layers (in the
    plain form the plan's rows, or the token list of each adapter)."""
    s = dict(_inputs(case, seed), case=case)
    step = case["mode"] == "step"
    if case["op"] == "route":
        if own and step:
            s["logits"].requires_grad_()
        return s
    if case["op"] == "lora":
        adapter = s.pop("adapter")
        s["adapter"] = torch.tensor(adapter, dtype=torch.int32, device="cuda")
        if own:
            s["plan"] = _kernels().token_plan(s["adapter"], case["L"])
        else:
            used = sorted(set(adapter) - {-1})
            s["tokens"] = [(a, torch.tensor([t for t, v in enumerate(adapter) if v == a], device="cuda")) for a in used]
        # base, the frozen projection's output, passes the incoming gradient on
        # as it is: nothing to compute or return
        leaves = ("x", "down", "up")
    else:
        ids = s.pop("ids")
        if own:
            s["plan"] = _kernels().token_plan(ids, case["E"], _MULTIPLE)
        else:
            s["rows"], s["src"] = _plan(ids, case["E"], _MULTIPLE)[:2]
        leaves = ("x",) if case["op"] == "dispatch" else ("y", "weights")
    if own and step:
        for name in leaves:
            s[name].requires_grad_()
    return s


# --- one pass ---------------------------------------------------------------


def run(state):
    """One pass through the case's operator."""
    return (_run_own if own else _PLAIN[state["case"]["op"]])(state)


def _run_own(s):
    kernels, case = _kernels(), s["case"]
    op, step = case["op"], case["mode"] == "step"
    if op == "route":
        s["logits"].grad = None
        r = kernels.moe_route(s["logits"], case["k"], normalize=case["normalize"], multiple_of=_MULTIPLE)
        out = (r.weights, r.ids, r.plan.rows, r.plan.src, r.plan.counts, r.plan.offs, r.balance_loss, r.z_loss)
        if step:
            torch.autograd.backward((r.weights, r.balance_loss, r.z_loss), (s["g_weights"], s["g_balance"], s["g_z"]))
            out += (s["logits"].grad,)
        return out
    if op == "dispatch":
        s["x"].grad = None
        out = kernels.moe_dispatch(s["x"], s["plan"])
        if not step:
            return out
        out.backward(s["g"])
        return out, s["x"].grad
    if op == "combine":
        s["y"].grad = s["weights"].grad = None
        out = kernels.moe_combine(s["y"], s["weights"], s["plan"])
        if not step:
            return out
        out.backward(s["g"])
        return out, s["y"].grad, s["weights"].grad
    s["x"].grad = s["down"].grad = s["up"].grad = None
    out = kernels.lora_grouped_mm(s["x"], s["down"], s["up"], s["plan"], scales=s["scales"], base=s["base"])
    if not step:
        return out
    out.backward(s["g"])
    return out, s["x"].grad, s["down"].grad, s["up"].grad


def _plan(ids, E, multiple):
    """(rows, src, counts, offs) of expert ids (T, k), -1 for no expert: the
    entries sorted by expert, in order, each group padded to the multiple."""
    flat = ids.reshape(-1)
    n = flat.numel()
    counts = (flat.unsqueeze(1) == torch.arange(E, device=ids.device, dtype=ids.dtype)).sum(dim=0)
    ends = ((counts + multiple - 1) // multiple * multiple).cumsum(dim=0)
    sizes = torch.diff(ends, prepend=ends.new_zeros(1))
    key = torch.where(flat < 0, E, flat)
    order = key.argsort(stable=True)                        # entries, dropped ones last
    first = torch.cat((counts.cumsum(dim=0) - counts, counts.sum().reshape(1)))
    start = torch.cat((ends - sizes, ends.new_zeros(1)))
    skey = key[order].long()
    row = start[skey] + torch.arange(n, device=ids.device) - first[skey]
    row = torch.where(skey == E, -1, row)
    rows = torch.empty_like(flat)
    rows[order] = row.to(torch.int32)
    cap = _capacity(n, E, multiple)
    src = torch.full((cap + 1,), -1, dtype=torch.int32, device=ids.device)
    src[torch.where(skey == E, cap, row)] = order.to(torch.int32)       # the last place takes the dropped ones
    return rows.reshape(ids.shape), src[:cap], counts.to(torch.int32), ends.to(torch.int32)


def _plain_route(s):
    case, k = s["case"], s["case"]["k"]
    E = case["E"]
    l = s["logits"].float()
    live = l.amax(dim=1) > float("-inf")
    m = torch.where(live, l.amax(dim=1), 0.0)
    e = (l - m.unsqueeze(1)).exp()
    z = torch.where(live, e.sum(dim=1), 1.0)
    p = e / z.unsqueeze(1)
    lse = torch.where(live, m + z.log(), 0.0)
    top, ids = l.sort(dim=1, descending=True, stable=True)
    ids, open_ = ids[:, :k], top[:, :k] > float("-inf")
    raw = torch.where(open_, p.gather(1, ids), 0.0)
    total = raw.sum(dim=1, keepdim=True)
    total = torch.where(live.unsqueeze(1), total, 1.0)
    weights = raw / total if case["normalize"] else raw
    chosen = torch.where(open_, ids, -1).to(torch.int32)
    rows, src, counts, offs = _plan(chosen, E, _MULTIPLE)
    n = live.sum().clamp_min(1).float()
    share = counts.float() / (n * k)
    balance = E * (share * (p.sum(dim=0) / n)).sum()
    z_loss = (lse * lse).sum() / n
    out = (weights, chosen, rows, src, counts, offs, balance, z_loss)
    if case["mode"] != "step":
        return out
    gw = torch.where(open_, s["g_weights"], 0.0)
    if case["normalize"]:
        own_part = weights * (gw - (weights * gw).sum(dim=1, keepdim=True))
        gp = torch.zeros_like(p)
    else:
        own_part = None
        gp = torch.zeros_like(p).scatter(1, ids, gw)
    gp = gp + s["g_balance"] * E * share / n
    gl = p * (gp - (p * gp).sum(dim=1, keepdim=True)) + p * (2 * s["g_z"] * lse / n).unsqueeze(1)
    if own_part is not None:
        gl = gl.scatter_add(1, ids, own_part)
    return out + (gl.to(s["logits"].dtype),)


def _gather_rows(t, index):
    """Rows of t, zeros where the index is -1."""
    return torch.where(index.unsqueeze(-1) >= 0, t[index.clamp_min(0).long()], torch.zeros((), dtype=t.dtype,
                                                                                         device=t.device))


def _plain_dispatch(s):
    k = s["case"]["k"]
    token = torch.where(s["src"] >= 0, s["src"] // k, -1)
    out = _gather_rows(s["x"], token)
    if s["case"]["mode"] != "step":
        return out
    gx = _gather_rows(s["g"], s["rows"][:, 0]).float()
    for j in range(1, k):
        gx = gx + _gather_rows(s["g"], s["rows"][:, j]).float()
    return out, gx.to(s["x"].dtype)


def _plain_combine(s):
    k, w = s["case"]["k"], s["weights"]
    out = torch.zeros((w.shape[0], s["y"].shape[1]), device=w.device)
    for j in range(k):
        out = out + w[:, j:j + 1] * _gather_rows(s["y"], s["rows"][:, j]).float()
    out = out.to(s["y"].dtype)
    if s["case"]["mode"] != "step":
        return out
    g = s["g"].float()
    token = torch.where(s["src"] >= 0, s["src"] // k, -1)
    gate = torch.where(s["src"] >= 0, w.reshape(-1)[s["src"].clamp_min(0).long()], 0.0)
    gy = (_gather_rows(g, token) * gate.unsqueeze(1)).to(s["y"].dtype)
    gw = torch.stack([(g * _gather_rows(s["y"], s["rows"][:, j]).float()).sum(dim=1) for j in range(k)], dim=1)
    return out, gy, gw


def _plain_lora(s):
    case = s["case"]
    x, down, up, sc = s["x"], s["down"], s["up"], s["scales"]
    out = s["base"].float()
    if case["mode"] == "fwd" and case["T"] <= 256:
        # few tokens: every token's own adapter, all at once
        a = s["adapter"].clamp_min(0).long()
        scale = torch.where(s["adapter"] >= 0, sc[a], 0.0)
        h = torch.bmm(down[a].float(), x.float().unsqueeze(2))
        delta = torch.bmm(h.transpose(1, 2).contiguous(), up[a].float()).squeeze(1)
        return (out + delta * scale.unsqueeze(1)).to(x.dtype)
    xf, h = x.float(), {}
    for a, tok in s["tokens"]:
        h[a] = xf[tok] @ down[a].float().t()
        out[tok] += sc[a] * (h[a] @ up[a].float())
    out = out.to(x.dtype)
    if case["mode"] == "fwd":
        return out
    g = s["g"].float()
    gx, gdown, gup = torch.zeros_like(xf), torch.zeros_like(down), torch.zeros_like(up)
    for a, tok in s["tokens"]:
        ga = g[tok] * sc[a]
        u = ga @ up[a].float().t()
        gx[tok] = u @ down[a].float()
        gdown[a] = (u.t() @ xf[tok]).to(down.dtype)
        gup[a] = (h[a].t() @ ga).to(up.dtype)
    return out, gx.to(x.dtype), gdown, gup


_PLAIN = {"route": _plain_route, "dispatch": _plain_dispatch, "combine": _plain_combine, "lora": _plain_lora}


# --- what a case takes and gives --------------------------------------------


def work(case):
    """Bytes and operations the path cannot do without: each input read once,
    each output written once, two operations per multiply-add."""
    T, b, step = case["T"], _BYTES[case["dtype"]], case["mode"] == "step"
    if case["op"] == "lora":
        r, K, N = case["r"], case["K"], case["N"]
        used = len(set(_adapters(case, 1)) - {-1})
        byt = b * (T * (K + 2 * N) + used * r * (K + N))
        if step:        # gradient in; gradients of x, down and up out
            byt += b * (T * (K + N) + case["L"] * r * (K + N))
        return {"bytes": byt, "flops": 2 * T * r * (K + N) * (3 if step else 1)}
    k, E = case["k"], case["E"]
    M = _capacity(T * k, E, _MULTIPLE)
    if case["op"] == "route":
        byt = T * E * b + 12 * T * k + 4 * M + 8 * E
        if step:
            byt += T * E * b + 4 * T * k
        return {"bytes": byt, "flops": (10 if step else 5) * T * E}
    H = case["H"]
    plan = 4 * T * k
    if case["op"] == "dispatch":
        one = b * H * (T + M) + plan
        return {"bytes": one * (2 if step else 1), "flops": T * k * H if step else 0}
    byt = b * H * (T * k + T) + 2 * plan
    if step:
        byt += b * H * (T + M) + plan
    return {"bytes": byt, "flops": 2 * T * k * H * (3 if step else 1)}


def _exact_plan(chosen, E):
    """The plan from its definition, group by group on the host."""
    flat = chosen.reshape(-1).tolist()
    groups = [[] for _ in range(E)]
    for i, e in enumerate(flat):
        if e >= 0:
            groups[e].append(i)
    rows, src, ends, at = [-1] * len(flat), [-1] * _capacity(len(flat), E, _MULTIPLE), [], 0
    for g in groups:
        for n, i in enumerate(g):
            rows[i] = at + n
            src[at + n] = i
        at += -(-len(g) // _MULTIPLE) * _MULTIPLE
        ends.append(at)

    def t(v):
        return torch.tensor(v, dtype=torch.int32, device=chosen.device)

    return t(rows).reshape(chosen.shape), t(src), t([len(g) for g in groups]), t(ends)


def _exact_route(case, s):
    E, k = case["E"], case["k"]
    l = s["logits"].double().requires_grad_()
    live = torch.isfinite(l).any(dim=1)
    safe = torch.where(live.unsqueeze(1), l, 0.0)
    p = torch.where(live.unsqueeze(1), torch.softmax(safe, dim=1), 0.0)
    lse = torch.where(live, torch.logsumexp(safe, dim=1), 0.0)
    # the k largest, one after the other; argmax of the first maximum
    left, ids = s["logits"].float().clone(), []
    for _ in range(k):
        best = left.amax(dim=1, keepdim=True)
        at = (left == best).to(torch.int8).argmax(dim=1)
        ids.append(torch.where(best[:, 0] > float("-inf"), at, -1))
        left.scatter_(1, at.unsqueeze(1), float("-inf"))
    chosen = torch.stack(ids, dim=1).to(torch.int32)
    raw = torch.where(chosen >= 0, p.gather(1, chosen.clamp_min(0).long()), 0.0)
    weights = raw / torch.where(live, raw.sum(dim=1), 1.0).unsqueeze(1) if case["normalize"] else raw
    rows, src, counts, offs = _exact_plan(chosen, E)
    n = max(1, int(live.sum()))
    balance = E * ((counts.double() / (n * k)) * (p.sum(dim=0) / n)).sum()
    z_loss = (lse ** 2).sum() / n
    out = (weights.detach(), chosen, rows, src, counts, offs, balance.detach(), z_loss.detach())
    if case["mode"] != "step":
        return out
    objective = (weights * s["g_weights"].double()).sum() + balance * s["g_balance"].double() + z_loss * s["g_z"].double()
    objective.backward()
    return out + (l.grad,)


def exact(case, seed):
    """What run() returns, from the operators' definitions in 64 bits."""
    s = _inputs(case, seed)
    step = case["mode"] == "step"
    if case["op"] == "route":
        return _exact_route(case, s)
    if case["op"] == "lora":
        x, g = s["x"].double(), s["g"].double() if step else None
        out = s["base"].double()
        adapter = torch.tensor(s["adapter"], device="cuda")
        gx = torch.zeros_like(x) if step else None
        gdown = torch.zeros(s["down"].shape, dtype=torch.float64, device="cuda") if step else None
        gup = torch.zeros(s["up"].shape, dtype=torch.float64, device="cuda") if step else None
        for a in range(case["L"]):
            tok = torch.nonzero(adapter == a)[:, 0]
            if tok.numel() == 0:
                continue
            down, up, sc = s["down"][a].double(), s["up"][a].double(), s["scales"][a].double()
            full = sc * (down.t() @ up)                     # the adapter as one K x N matrix
            if step or case["r"] * 4 > tok.numel():
                out[tok] += sc * ((x[tok] @ down.t()) @ up)
            else:
                out[tok] += x[tok] @ full
            if step:
                gx[tok] = g[tok] @ full.t()
                outer = sc * (x[tok].t() @ g[tok])          # gradient of the K x N matrix, over its factors
                gdown[a], gup[a] = up @ outer.t(), down @ outer
        return (out, gx, gdown, gup) if step else out
    T, H, k = case["T"], case["H"], case["k"]
    rows, src, _, _ = _exact_plan(s["ids"], case["E"])
    valid = (src >= 0).nonzero()[:, 0]
    entry = src[valid].long()
    token = entry // k
    if case["op"] == "dispatch":
        out = torch.zeros((src.numel(), H), dtype=s["x"].dtype, device="cuda")
        out[valid] = s["x"][token]
        out = out.double()
        if not step:
            return out
        return out, torch.zeros((T, H), dtype=torch.float64, device="cuda").index_add_(0, token, s["g"][valid].double())
    w = s["weights"].double().reshape(-1)[entry].unsqueeze(1)
    y = s["y"][valid].double()
    out = torch.zeros((T, H), dtype=torch.float64, device="cuda").index_add_(0, token, w * y)
    if not step:
        return out
    g = s["g"].double()[token]
    gy = torch.zeros((src.numel(), H), dtype=torch.float64, device="cuda")
    gy[valid] = w * g
    gw = torch.zeros((T * k,), dtype=torch.float64, device="cuda")
    gw[entry] = (g * y).sum(dim=1)
    return out, gy, gw.reshape(T, k)
