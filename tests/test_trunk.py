"""The gated residual step with its norms (nvp_amd.trunk) against a plain 64-bit evaluation, its refusals, and the conditioning operators together.

Tolerances.  e = 2^-24.  A sum over a row takes at most 8 additions in a lane, 6 across a wave and 15 across waves (< 30 e), so 1 / rms is off by < 20 e of
itself plus what its input is off by.  Every result is a sum of products of such numbers; counted along the longest chain (norm, gate, y, second norm, two
means, the result) fewer than 200 roundings are made, each of at most e of a number no larger than the same expression with every term made
positive, M.  y enters the second norm with its own error, which counts K = |A| / |y| times (A: y with its two terms made positive).  So
|got - exact| <= 200 K e M + eps / 2 |exact|; sums over R rows add at most R + 64 roundings: (200 K + R + 64) e M."""
import ctypes

import pytest
import torch

from nvp_amd import _lib as L
from nvp_amd import codes, quantize, trunk

F32, B16, F16 = torch.float32, torch.bfloat16, torch.float16
E = 2.0 ** -24


def dev():
    return torch.device("cuda:0")


def plain(leaf, scale, act, eps):
    """outputs (y, u) in the leaves' type (float64), from the definition"""
    rms = lambda v: torch.sqrt(torch.mean(v * v, -1, keepdim=True) + eps)      # noqa: E731
    y, outs = leaf["x"], []
    if "h" in leaf:
        add = scale * leaf["h"] / rms(leaf["h"]) * leaf["post"]
        if "gate" in leaf:
            add = add * (torch.sigmoid(leaf["gate"]) if act == "sigmoid" else leaf["gate"])
        y = y + add
        outs.append(y)
    if "next" in leaf:
        outs.append(y / rms(y) * leaf["next"])
    return outs


def magnitudes(leaf, seeds, scale, act, eps):
    """M of every output and gradient (rows flattened), and K"""
    d = leaf["x"].shape[-1]
    x = leaf["x"].abs().reshape(-1, d)
    rows = x.shape[0]
    seeds = [s.abs().reshape(-1, d) for s in seeds]
    out, grad = [], {}
    full = plain(leaf, scale, act, eps)
    A, K, r2 = x, 1.0, None
    if "h" in leaf:
        h = leaf["h"].reshape(-1, d)
        r1 = 1 / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
        n = h.abs() * r1
        if "gate" in leaf:
            g = leaf["gate"].expand(leaf["x"].shape).reshape(-1, d)
            a, da = (torch.sigmoid(g), torch.sigmoid(g) * (1 - torch.sigmoid(g))) if act == "sigmoid" else (g.abs(), torch.ones_like(g))
        else:
            a, da = torch.ones_like(n), torch.zeros_like(n)
        p = leaf["post"].abs()
        A = x + abs(scale) * a * n * p
        out.append(A)
    m = seeds[0] if "h" in leaf else torch.zeros_like(x)
    if "next" in leaf:
        y = (full[0] if "h" in leaf else leaf["x"]).reshape(-1, d)
        r2 = 1 / torch.sqrt((y * y).mean(-1, keepdim=True) + eps)
        K = float((A.norm(dim=1) / (y.norm(dim=1) + 1e-300)).max())
        w, du = leaf["next"].abs(), seeds[-1]
        v = A * r2
        out.append(v * w)
        m = m + r2 * (du * w + v * (du * w * v).mean(-1, keepdim=True))
        grad["next"] = (du * v).sum(0)
    grad["x"] = m
    if "h" in leaf:
        dn = abs(scale) * a * p * m
        grad["h"] = r1 * (dn + n * (dn * n).mean(-1, keepdim=True))
        grad["post"] = (abs(scale) * a * n * m).sum(0)
        if "gate" in leaf:
            grad["gate"] = (abs(scale) * n * p * da * m).reshape(leaf["gate"].numel() // d, -1, d).sum(1)
    return out, grad, max(K, 1.0), rows


def within(got, want, m, roundings, what):
    half = torch.finfo(got.dtype).eps / 2
    got, want = got.detach().double().cpu().reshape(m.shape), want.detach().cpu().reshape(m.shape)
    err = (got - want).abs()
    tol = roundings * E * m.cpu() * (1 + half) + half * want.abs() + torch.finfo(F32).tiny
    if half > E:
        tol = tol + torch.finfo(B16).tiny + (2.0 ** -25 if half == torch.finfo(F16).eps / 2 else 0)      # below fp16's normal numbers: half of 2^-24
    assert bool((err <= tol).all()), f"{what}: {float((err - tol).max())} over the tolerance, error {float(err.max())}"


def make(shape, dtype, wdtype, form, gate, seed):
    g = torch.Generator().manual_seed(seed)
    d = shape[-1]
    r = lambda *s, std=1.0, mean=0.0, t=dtype: (torch.randn(s, generator=g) * std + mean).to(t).to(dev())      # noqa: E731
    leaf = {"x": r(*shape, std=1.5)}
    if form != "first":
        leaf["h"] = r(*shape, std=0.7)
        leaf["post"] = r(d, std=0.2, mean=1.0, t=wdtype)
        if gate is not None:
            leaf["gate"] = r(*gate)
    if form != "last":
        leaf["next"] = r(d, std=0.2, mean=1.0, t=wdtype)
    seeds = [r(*shape) for _ in range((form != "first") + (form != "last"))]
    return leaf, seeds


def call(leaf, scale, act, eps):
    if "h" not in leaf:
        return [trunk.pre_norm(leaf["x"], leaf["next"], eps)]
    r = trunk.gated_residual(leaf["x"], leaf["h"], leaf.get("gate"), leaf["post"], leaf.get("next"), scale, act, eps)
    return list(r) if "next" in leaf else [r]


def check(leaf, seeds, scale, act, eps=1e-6):
    mine = {k: v.detach().clone().requires_grad_(True) for k, v in leaf.items()}
    outs = call(mine, scale, act, eps)
    names = list(mine)
    grads = dict(zip(names, torch.autograd.grad(outs, [mine[k] for k in names], seeds)))
    ref = {k: v.detach().double().cpu().requires_grad_(True) for k, v in leaf.items()}
    want = plain(ref, scale, act, eps)
    sd = [s.double().cpu() for s in seeds]
    wgrads = dict(zip(names, torch.autograd.grad(want, [ref[k] for k in names], sd)))
    with torch.no_grad():
        mo, mg, K, rows = magnitudes({k: v.detach() for k, v in ref.items()}, sd, scale, act, eps)
    for o, w, m, s in zip(outs, want, mo, ("y", "u")):
        assert o.dtype == leaf["x"].dtype and o.shape == leaf["x"].shape
        within(o, w, m, 200 * K, "y" if "h" in leaf and s == "y" else "u")
    for k in names:
        assert grads[k].dtype == leaf[k].dtype and grads[k].shape == leaf[k].shape
        summed = k in ("post", "next") or (k == "gate" and leaf["gate"].numel() < leaf["x"].numel())
        within(grads[k], wgrads[k], mg[k], 200 * K + (rows + 64 if summed else 0), "d" + k)
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(call(leaf, scale, act, eps), outs))            # without a backward pass: the same bits
    again = torch.autograd.grad(call(mine, scale, act, eps), [mine[k] for k in names], seeds)
    assert all(torch.equal(a, grads[k]) for a, k in zip(again, names))


# ---- on the host -------------------------------------------------------------------------------------------------------------------------------
def test_refusals_on_the_host():
    x, w = torch.zeros(2, 3, 8), torch.ones(8)
    with pytest.raises(RuntimeError, match="HIP device"):
        trunk.pre_norm(x, w)
    with pytest.raises(RuntimeError, match="HIP device"):
        trunk.gated_residual(x, x, None, w)
    with pytest.raises(RuntimeError, match="a weight"):
        trunk.pre_norm(x, torch.ones(7))
    with pytest.raises(RuntimeError, match="a weight"):
        trunk.pre_norm(x.half(), w.bfloat16())
    with pytest.raises(RuntimeError, match="a weight"):
        trunk.pre_norm(x, w.half())
    with pytest.raises(RuntimeError, match="of one type"):
        trunk.gated_residual(x.half(), x.half(), None, w, w.half())
    with pytest.raises(RuntimeError, match="1 <= D <= 8192"):
        trunk.pre_norm(torch.zeros(2, 8200), torch.ones(8200))
    with pytest.raises(RuntimeError, match="1 <= D <= 8192"):
        trunk.pre_norm(torch.zeros(2, 0), torch.ones(0))
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        trunk.pre_norm(x.double(), w.double())
    with pytest.raises(RuntimeError, match="h must be like x"):
        trunk.gated_residual(x, x[:1], None, w)
    with pytest.raises(RuntimeError, match="h must be like x"):
        trunk.gated_residual(x, x.half(), None, w)
    for bad in (torch.zeros(2, 1, 7), torch.zeros(1, 3, 8), torch.zeros(3, 1, 8), torch.zeros(2, 3, 8, dtype=torch.float16), torch.zeros(1, 2, 3, 8), torch.tensor(1.0)):
        with pytest.raises(RuntimeError, match="a gate for x"):
            trunk.gated_residual(x, x, bad, w)
    with pytest.raises(RuntimeError, match="gate_act"):
        trunk.gated_residual(x, x, x, w, gate_act="tanh")
    with pytest.raises(RuntimeError, match="eps"):
        trunk.pre_norm(x, w, eps=-1.0)
    with pytest.raises(RuntimeError, match="eps"):
        trunk.pre_norm(x, w, eps=float("nan"))
    with pytest.raises(RuntimeError, match="scale"):
        trunk.gated_residual(x, x, None, w, scale=float("inf"))
    with pytest.raises(ValueError):
        trunk.Trunk(8193, 1)
    for gate in (x, torch.zeros(2, 1, 8), torch.zeros(1, 1, 8), torch.zeros(1, 8), torch.zeros(8)):      # taken: what is refused is the device
        with pytest.raises(RuntimeError, match="HIP device"):
            trunk.gated_residual(x, x, gate, w, w)


def test_entry_points_refuse_bad_arguments_without_a_device():
    lib, d = L.load(), ctypes.c_void_p(64)                             # never dereferenced

    def args(**kw):
        v = dict(x=64, h=64, gate=64, post=64, next=64, rows=6, gate_rows=3, dim=8, type=1, weight_type=0, gate_act=1, scale=1.0, eps=1e-6)
        v.update(kw)
        return ctypes.byref(L.Residual(*[v[f[0]] for f in L.Residual._fields_]))
    need = lib.nvp_residual_bwd_workspace_bytes(args())
    assert need > 0
    for kw in (dict(rows=-1), dict(dim=0), dict(type=3), dict(weight_type=2), dict(gate_act=2), dict(gate_rows=4), dict(gate_rows=0), dict(gate_rows=12), dict(eps=-1.0),
               dict(eps=float("nan")), dict(h=None), dict(post=None), dict(h=None, post=None), dict(h=None, post=None, gate=None, next=None)):
        assert lib.nvp_residual_bwd_workspace_bytes(args(**kw)) == L.ERR_BADARG, kw
        assert lib.nvp_residual_fwd(args(**kw), d, d, None, None) == L.ERR_BADARG, kw
    assert lib.nvp_residual_fwd(args(dim=8193), d, d, None, None) == L.ERR_UNSUPPORTED
    assert lib.nvp_residual_fwd(args(x=None), d, d, None, None) == L.ERR_BADARG
    assert lib.nvp_residual_fwd(args(), None, d, None, None) == L.ERR_BADARG and lib.nvp_residual_fwd(args(), d, None, None, None) == L.ERR_BADARG
    assert lib.nvp_residual_fwd(args(rows=0), None, None, None, None) == 0
    assert lib.nvp_residual_bwd(args(), None, d, d, d, d, d, d, d, d, need, None) == L.ERR_BADARG                  # no stats
    assert lib.nvp_residual_bwd(args(), d, d, d, d, d, d, d, d, d, need - 1, None) == L.ERR_BADARG
    assert lib.nvp_residual_bwd(args(next=None), d, d, d, d, d, d, d, None, d, need, None) == L.ERR_BADARG         # du without u
    assert lib.nvp_residual_bwd(args(gate=None), d, d, d, d, d, d, d, d, d, need, None) == L.ERR_BADARG            # dgate without a gate


# ---- on the device -----------------------------------------------------------------------------------------------------------------------------
TYPES = [(F32, F32), (B16, F32), (B16, B16), (F16, F32), (F16, F16)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,wdtype", TYPES)
@pytest.mark.parametrize("form", ["both", "first", "last"])
@pytest.mark.parametrize("rows,d", [(1, 1), (2, 3), (5, 16), (37, 114), (40, 128), (33, 228), (7, 500), (9, 1000), (3, 2048), (2, 4096), (5, 4099), (2, 8192)])
def test_residual(rows, d, form, dtype, wdtype):
    leaf, seeds = make((rows, d), dtype, wdtype, form, (rows, d) if rows % 2 else None, rows * 10000 + d)
    check(leaf, seeds, 0.75, "sigmoid" if d % 2 == 0 else None, eps=1e-3 if d < 16 else 1e-6)


@pytest.mark.gpu
@pytest.mark.parametrize("shape,gate", [((4, 6, 32), (4, 1, 32)), ((4, 6, 32), (1, 1, 32)), ((4, 6, 32), (32,)), ((3, 2, 5, 40), (3, 2, 1, 40)), ((3, 2, 5, 40), (3, 1, 1, 40)),
                                        ((2, 4000, 24), (2, 1, 24)), ((700, 3, 130), (700, 1, 130)), ((5000, 2, 8), (5000, 1, 8)), ((2, 1500, 1030), (2, 1, 1030)),
                                        ((1, 900, 4096), (1, 1, 4096)), ((6, 1, 64), (6, 1, 64))])
@pytest.mark.parametrize("act", [None, "sigmoid"])
def test_residual_shared_gates(shape, gate, act):
    """A gate row for several rows: its gradient is summed within a unit, over pieces, or over everything."""
    for form in ("both", "last"):
        leaf, seeds = make(shape, F32, F32, form, gate, sum(shape))
        check(leaf, seeds, -0.5, act)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,d", [(20000, 16), (9000, 300), (5000, 640), (3000, 2050)])
def test_residual_many_rows(rows, d):
    leaf, seeds = make((rows, d), B16, F32, "both", (rows, d), rows)
    check(leaf, seeds, 1.0, "sigmoid")


@pytest.mark.gpu
def test_residual_against_differences():
    """<grad, z> against the difference quotient of the kernel's own forward along z.  The quotient of the 64-bit function at the same step says how far a
    quotient is from the derivative (T); the kernel's forward is off by at most the forward tolerance at either end, the gradients by theirs."""
    eps, scale, act, step = 1e-6, 0.8, "sigmoid", 2.0 ** -6
    leaf, seeds = make((6, 5, 48), F32, F32, "both", (6, 1, 48), 3)
    g = torch.Generator().manual_seed(9)
    z = {k: (torch.randn(v.shape, generator=g) * 16).round().div(16).to(dev()) for k, v in leaf.items()}
    mine = {k: v.clone().requires_grad_(True) for k, v in leaf.items()}
    grads = dict(zip(mine, torch.autograd.grad(call(mine, scale, act, eps), list(mine.values()), seeds)))
    dot = sum(float((grads[k].double() * z[k].double()).sum()) for k in grads)

    def loss(f, sign, t):
        moved = {k: (leaf[k] + sign * step * z[k]).to(t) for k in leaf}
        with torch.no_grad():
            return sum(float((o.double() * s.double()).sum()) for o, s in zip(f(moved), seeds)), moved
    kp, at_p = loss(lambda v: call(v, scale, act, eps), 1, F32)
    km, at_m = loss(lambda v: call(v, scale, act, eps), -1, F32)
    pf = lambda v: plain(v, scale, act, eps)      # noqa: E731
    wide = lambda v: [o for o in pf({k: t.double() for k, t in v.items()})]      # noqa: E731
    pp, pm = (sum(float((o * s.double()).sum()) for o, s in zip(wide(v), seeds)) for v in (at_p, at_m))
    ref = {k: v.double().requires_grad_(True) for k, v in leaf.items()}
    wgrads = torch.autograd.grad(pf(ref), list(ref.values()), [s.double() for s in seeds])
    true = sum(float((w * z[k].double()).sum()) for k, w in zip(ref, wgrads))
    far = abs((pp - pm) / (2 * step) - true)
    fwd, grad = 0.0, 0.0
    for v in (at_p, at_m):
        mo, _, K, rows = magnitudes({k: t.double().cpu() for k, t in v.items()}, [s.double().cpu() for s in seeds], scale, act, eps)
        fwd += sum(float((200 * K * E * m * s.double().cpu().abs().reshape(m.shape)).sum()) for m, s in zip(mo, seeds))
    _, mg, K, rows = magnitudes({k: t.double().cpu() for k, t in leaf.items()}, [s.double().cpu() for s in seeds], scale, act, eps)
    for k in grads:
        grad += float(((200 * K + rows + 64) * E * mg[k] * z[k].double().cpu().abs().reshape(mg[k].shape)).sum())
    assert far < 0.05 * abs(true) + 1.0                                  # the step is small enough for the quotient to mean something
    assert abs((kp - km) / (2 * step) - dot) <= far + fwd / (2 * step) + grad


@pytest.mark.gpu
def test_residual_partial_gradients_and_unused_outputs():
    leaf, seeds = make((4, 9, 72), F32, F32, "both", (4, 1, 72), 5)
    full = {k: v.clone().requires_grad_(True) for k, v in leaf.items()}
    y, u = call(full, 1.0, "sigmoid", 1e-6)
    for outs, sd in (([y], seeds[:1]), ([u], seeds[1:])):
        zero = [s if o is outs[0] else torch.zeros_like(s) for o, s in zip((y, u), seeds)]
        a = torch.autograd.grad(outs, list(full.values()), sd, retain_graph=True, allow_unused=True)
        b = torch.autograd.grad([y, u], list(full.values()), zero, retain_graph=True)
        assert all(torch.equal(p if p is not None else torch.zeros_like(q), q) for p, q in zip(a, b))
    every = torch.autograd.grad([y, u], list(full.values()), seeds)
    for only in leaf:
        one = {k: v.clone().requires_grad_(k == only) for k, v in leaf.items()}
        g, = torch.autograd.grad(call(one, 1.0, "sigmoid", 1e-6), [one[only]], seeds)
        assert torch.equal(g, every[list(leaf).index(only)]), only
    # the same tensor as x and h, and as the gate: gradients add up
    x = leaf["x"].clone().requires_grad_(True)
    y2, u2 = trunk.gated_residual(x, x, x, leaf["post"], leaf["next"])
    g, = torch.autograd.grad([y2, u2], x, seeds)
    xs = [leaf["x"].clone().requires_grad_(True) for _ in range(3)]
    y3, u3 = trunk.gated_residual(*xs, leaf["post"], leaf["next"])
    parts = torch.autograd.grad([y3, u3], xs, seeds)
    # autograd adds the three parts in its own order: two fp32 additions, each off by at most 2^-24 of the parts' sizes
    assert bool(((g - (parts[0] + parts[1] + parts[2])).abs() <= 4 * E * (parts[0].abs() + parts[1].abs() + parts[2].abs())).all())


@pytest.mark.gpu
def test_residual_zero_rows_and_non_finite_values():
    for eps in (1e-6, 1e-30):
        leaf, seeds = make((6, 200), F32, F32, "both", (6, 200), 11)
        leaf["h"][2] = 0                                                    # 1 / rms = eps^-1/2
        mine = {k: v.clone().requires_grad_(True) for k, v in leaf.items()}
        y, u = call(mine, 1.0, None, eps)
        assert torch.equal(y[2], leaf["x"][2])
        g = torch.autograd.grad([y, u], list(mine.values()), seeds)
        assert all(bool(t.isfinite().all()) for t in g)
    leaf["x"][2] = 0
    y, u = call(leaf, 1.0, None, 1e-6)
    assert not y[2].any() and not u[2].any()
    bad = {k: v.clone() for k, v in leaf.items()}
    bad["x"][1, 3], bad["h"][3, 0], bad["gate"][5, 199] = float("nan"), float("inf"), float("nan")
    y, u = call(bad, 1.0, None, 1e-6)
    ok = [0, 2, 4]
    want = call(leaf, 1.0, None, 1e-6)
    assert torch.equal(y[ok], want[0][ok]) and torch.equal(u[ok], want[1][ok])
    assert bool(u[1].isnan().all()) and bool(u[5].isnan().all()) and bool(y[3, 0].isnan())
    saturated = {k: v.clone() for k, v in leaf.items()}
    saturated["gate"][0], saturated["gate"][1] = 1e4, -1e4
    y, _ = call(saturated, 1.0, "sigmoid", 1e-6)
    assert torch.equal(y[1], leaf["x"][1]) and bool(y.isfinite().all())


@pytest.mark.gpu
def test_residual_strides_alignment_and_empty_batches():
    wide = torch.randn(5, 7, 300, device=dev())
    x, h = wide[..., 1:129], wide.transpose(0, 1)[..., 3:131].transpose(0, 1)
    gate, w = torch.randn(5, 1, 128, device=dev()), torch.randn(131, device=dev())
    a = trunk.gated_residual(x, h, gate, w[3:], w[1:129], 0.5, "sigmoid")
    b = trunk.gated_residual(x.contiguous(), h.contiguous(), gate, w[3:].clone(), w[1:129].clone(), 0.5, "sigmoid")
    for p, q in zip(a, b):                                                  # another vector width: sums in another order
        assert bool(((p - q).abs() <= 400 * E * (q.abs() + 4)).all())
    for shape in ((0, 64), (3, 0, 64)):
        x = torch.zeros(shape, device=dev(), requires_grad=True)
        h = torch.zeros(shape, device=dev(), requires_grad=True)
        g = torch.zeros(shape, device=dev(), requires_grad=True)
        ws = [torch.ones(64, device=dev(), requires_grad=True) for _ in range(2)]
        y, u = trunk.gated_residual(x, h, g, *ws)
        assert y.shape == u.shape == shape
        grads = torch.autograd.grad([y, u], [x, h, g, *ws], [torch.zeros_like(y)] * 2)
        assert all(not t.any() for t in grads) and grads[3].shape == (64,)


@pytest.mark.gpu
def test_residual_rows_do_not_depend_on_their_neighbours():
    leaf, _ = make((3000, 256), B16, F32, "both", (3000, 256), 2)
    y, u = call(leaf, 1.0, "sigmoid", 1e-6)
    part = {k: (v[1000:1003] if v.dim() == 2 else v) for k, v in leaf.items()}
    py, pu = call(part, 1.0, "sigmoid", 1e-6)
    assert torch.equal(py, y[1000:1003]) and torch.equal(pu, u[1000:1003])


@pytest.mark.gpu
def test_residual_captured_and_replayed():
    """Forward and backward inside one captured graph, replayed with other inputs and eager calls between the replays; a second graph beside it."""
    graphs = []
    for shape, gate in (((4, 300, 96), (4, 1, 96)), ((50, 2100), (50, 2100))):
        leaf, seeds = make(shape, B16, F32, "both", gate, 4)

        def step(leaf=leaf, seeds=seeds):
            mine = {k: v.detach().requires_grad_(True) for k, v in leaf.items()}
            outs = call(mine, 0.5, "sigmoid", 1e-6)
            return [o.detach() for o in outs] + list(torch.autograd.grad(outs, list(mine.values()), seeds))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        graphs.append((graph, got, step, leaf))
    for _ in range(3):
        for graph, got, step, leaf in graphs:
            leaf["x"].copy_(torch.randn(leaf["x"].shape, device=dev()))
            graph.replay()
        for graph, got, step, leaf in graphs:
            want = step()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---- the operators together ---------------------------------------------------------------------------------------------------------------------
def plain_trunk(t, x, params):
    rms = lambda v: torch.sqrt(torch.mean(v * v, -1, keepdim=True) + t.eps)      # noqa: E731
    lin = lambda n, k, v: v @ params[f"{n}.{k}.weight"].t() + params[f"{n}.{k}.bias"]      # noqa: E731
    u = x / rms(x) * params["norms.0"]
    for k in range(t.depth):
        h = lin("downs", k, torch.nn.functional.leaky_relu(lin("ups", k, u)))
        x = x + t.scale * torch.sigmoid(lin("gates", k, u)) * h / rms(h) * params[f"posts.{k}"]
        u = x / rms(x) * params[f"norms.{k + 1}"]
    return u


@pytest.mark.gpu
def test_codes_trunk_and_siren_together():
    """Codes of frames -> residual stack -> latent of the modulated SIREN, forward and backward; every gradient of the conditioning side against a 64-bit
    evaluation of the same stack, seeded with the gradient that the SIREN hands to its latent.  Two blocks are some 30 operators in a row, each off by
    fewer than 200 roundings of 2^-24 in the sense above: 30 * 200 * 2^-24 = 3.6e-4 of a tensor's norm at worst, were they all to add up."""
    from nvp_amd import modulation
    torch.manual_seed(0)
    d, frames, n = 114, 40, 900
    table, stack = codes.CodeTable(frames, d, scale=3.0).to(dev()), trunk.Trunk(d, 2, hidden=200).to(dev())
    with torch.no_grad():
        table.codes.normal_()
    net = modulation.SirenNet(dim_in=1, dim_hidden=128, dim_out=3, num_layers=3, w0_initial=30.)
    wrapper = modulation.SirenWrapper(net, latent_dim=d).to(dev())
    ids = torch.randint(0, frames, (n,), device=dev())
    latent = stack(table(ids))
    latent.retain_grad()
    out = wrapper(ids[:, None].float() / frames, latent)
    out.square().mean().backward()
    ref = {k: v.detach().double().cpu().requires_grad_(True) for k, v in stack.named_parameters()}
    rt = table.codes.detach().double().cpu().requires_grad_(True)
    want = plain_trunk(stack, 3.0 * rt[ids.cpu()], ref)
    tol = 3.6e-4
    rel = lambda a, b: float((a.detach().double().cpu() - b).norm() / b.norm())      # noqa: E731
    assert rel(latent, want.detach()) <= tol
    want.backward(latent.grad.double().cpu())
    assert rel(table.codes.grad, rt.grad) <= tol
    for k, p in stack.named_parameters():
        assert rel(p.grad, ref[k].grad) <= tol, k


@pytest.mark.gpu
def test_trunk_in_eight_bits():
    """to_8bit(): the same stack on linear8 - equal, bit for bit, to the operators called one by one, and captured as a whole."""
    torch.manual_seed(1)
    stack = trunk.Trunk(228, 2).to(dev())
    eight = stack.to_8bit()
    x = torch.randn(70, 228, device=dev())
    with torch.no_grad():
        got = eight(x)
        y, u = x, trunk.pre_norm(x, stack.norms[0])
        for k in range(2):
            q = {n: quantize.quantize_blocks(getattr(stack, n)[k].weight, 128) + (getattr(stack, n)[k].bias,) for n in ("ups", "downs", "gates")}
            h = quantize.linear8(torch.nn.functional.leaky_relu(quantize.linear8(u, *q["ups"])), *q["downs"])
            y, u = trunk.gated_residual(y, h, quantize.linear8(u, *q["gates"]), stack.posts[k], stack.norms[k + 1], stack.scale, "sigmoid")
        assert torch.equal(got, u)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            eight(x)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            cap = eight(x)
        for _ in range(3):
            x.normal_()
            graph.replay()
            want = eight(x)
            torch.cuda.synchronize()
            assert torch.equal(cap, want)
    with pytest.raises(NotImplementedError, match="inference-only"):
        eight(x.requires_grad_(True))
    other = trunk.Trunk(228, 2).to(dev()).to_8bit()
    other.load_state_dict(eight.state_dict())
    with torch.no_grad():
        assert torch.equal(other(x), eight(x))


@pytest.mark.gpu
def test_residual_is_differentiable_once_and_guards_what_it_saved():
    leaf, seeds = make((6, 40), F32, F32, "both", (6, 40), 3)
    mine = {k: v.requires_grad_(True) for k, v in leaf.items()}
    y, u = call(mine, 0.5, "sigmoid", 1e-6)
    g, = torch.autograd.grad((y, u), mine["x"], seeds, create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        g.sum().backward()
    y, u = call(mine, 0.5, "sigmoid", 1e-6)
    a = torch.autograd.grad((y, u), mine["h"], seeds, retain_graph=True)
    assert torch.equal(a[0], torch.autograd.grad((y, u), mine["h"], seeds)[0])
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad((y, u), mine["h"], seeds)
    h = mine["h"].detach().clone()
    y, u = trunk.gated_residual(mine["x"], h, None, mine["post"], mine["next"])
    h.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad((y, u), mine["x"], seeds)
    with pytest.raises(RuntimeError, match="HIP device"):
        trunk.gated_residual(mine["x"], mine["h"], None, mine["post"].cpu())


@pytest.mark.gpu
def test_residual_with_one_tensor_in_several_places():
    """x as its own block output and gate, one weight for both norms: the gradients of the places add up."""
    g = torch.Generator().manual_seed(5)
    x, w = torch.randn(33, 260, generator=g), 1 + 0.2 * torch.randn(260, generator=g)
    seeds = [torch.randn(33, 260, generator=g) for _ in range(2)]
    mx, mw = x.to(dev()).requires_grad_(True), w.to(dev()).requires_grad_(True)
    got = torch.autograd.grad(trunk.gated_residual(mx, mx, mx, mw, mw, 0.5, "sigmoid"), (mx, mw), [s.to(dev()) for s in seeds])
    one = [x.to(dev()).clone().requires_grad_(True) for _ in range(3)] + [w.to(dev()).clone().requires_grad_(True) for _ in range(2)]
    parts = torch.autograd.grad(trunk.gated_residual(*one, 0.5, "sigmoid"), one, [s.to(dev()) for s in seeds])
    for a, b in ((got[0], parts[:3]), (got[1], parts[3:])):
        s = sum(p.abs() for p in b)
        assert bool(((a - sum(b)).abs() <= 3 * E * 2 * s).all())           # at most two additions, in one order or another


@pytest.mark.gpu
def test_residual_offsets_past_32_bits():
    rows, d = 540_000, 4096
    r = lambda: torch.randn(rows, d, device=dev(), dtype=B16)      # noqa: E731
    leaf = {"x": r(), "h": r(), "gate": r(), "post": torch.rand(d, device=dev()) + 0.5, "next": torch.rand(d, device=dev()) + 0.5}
    seeds = [r(), r()]
    names = ("x", "h", "gate")

    def run(a, b):
        mine = {k: (v[a:b] if k in names else v).detach().requires_grad_(True) for k, v in leaf.items()}
        outs = call(mine, 0.5, "sigmoid", 1e-6)
        return [o.detach() for o in outs] + list(torch.autograd.grad(outs, [mine[k] for k in names], [s[a:b] for s in seeds]))
    full = run(0, rows)
    for a in (0, 524_250, rows - 70):                               # 524 288 rows: 2^31 values
        assert all(torch.equal(f[a:a + 70], p) for f, p in zip(full, run(a, a + 70)))


@pytest.mark.gpu
def test_trunk_under_autocast_keeps_the_stream_in_32_bits():
    torch.manual_seed(0)
    m = trunk.Trunk(64, 2).to(dev())
    x = torch.randn(30, 64, device=dev())
    want = m(x)
    with torch.autocast("cuda", dtype=B16):
        got = m(x)
    assert got.dtype == F32
    # two blocks of three products whose operands are rounded to bf16 (2^-9 each, relative): a few 2^-9 of the latent's size, which is 1
    assert float((got - want).square().mean().sqrt()) <= 2 ** -9 * 16
    got.sum().backward()
    assert all(p.grad is not None and bool(p.grad.isfinite().all()) for p in m.parameters())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,wdtype", TYPES)
@pytest.mark.parametrize("rows,d", [(3, 4097), (700, 4100), (5, 5000), (4, 6143), (2, 6144), (601, 6145), (3, 8191)])
def test_residual_wide_rows(rows, d, dtype, wdtype):
    for k, (form, gate) in enumerate((("both", (rows, d)), ("both", (1, d)), ("first", None), ("last", (rows, d)))):
        if rows > 100 and k:
            break
        leaf, seeds = make((rows, d), dtype, wdtype, form, gate, rows * 100 + d)
        check(leaf, seeds, 0.75, "sigmoid" if k % 2 == 0 else None)


@pytest.mark.gpu
def test_residual_wide_rows_do_not_depend_on_their_neighbours():
    for d in (4104, 5000, 6144, 8192):
        leaf, seeds = make((1500, d), B16, F32, "both", (1500, d), d)
        names = ("x", "h", "gate")

        def run(a, b):
            mine = {k: (v[a:b] if k in names else v).detach().requires_grad_(True) for k, v in leaf.items()}
            outs = call(mine, 0.5, "sigmoid", 1e-6)
            return [o.detach() for o in outs] + list(torch.autograd.grad(outs, [mine[k] for k in names], [s[a:b] for s in seeds]))
        full = run(0, 1500)
        assert all(torch.equal(f[1490:], p) for f, p in zip(full, run(1490, 1500)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,wdtype", TYPES)
@pytest.mark.parametrize("shape,gate", [((40, 228), (40, 228)), ((9, 115), (9, 115)), ((6, 50, 114), (6, 1, 114)), ((2, 1500, 130), (1, 1, 130)), ((3, 4100), (3, 4100)), ((2, 30, 8190), (2, 1, 8190)),
                                        ((3, 5003), (3, 5003)), ((2, 8190), (2, 8190)), ((3, 8192), (3, 8192))])
def test_residual_gates_far_open_and_far_closed(shape, gate, dtype, wdtype, monkeypatch):
    """A sigmoid's derivative is a (1 - a) whichever side a is near: every gradient to the tolerance above, of numbers down to 1e-13.  The 64-bit sigmoid is written
    out here, because autograd differentiates 1 / (1 + exp(-g)) without a difference, while torch.sigmoid's own backward has 1 - a (1e-3 off at 30, in 64 bits)."""
    monkeypatch.setattr(torch, "sigmoid", lambda g: 1 / (1 + torch.exp(-g)))
    leaf, seeds = make(shape, dtype, wdtype, "both", gate, sum(shape))
    g = torch.Generator().manual_seed(1)
    leaf["gate"] = (torch.rand(gate, generator=g) * 60 - 30).to(dtype).to(dev())
    check(leaf, seeds, 0.75, "sigmoid")


@pytest.mark.gpu
def test_residual_sigmoid_in_32_bits_far_from_zero():
    """y = scale * sigmoid(g) * n * post with x = 0: a chain of products, so the whole error is relative.  Roundings of 2^-24, counted as half ulps: the norm n < 20 (above) + 1 + 1
    (its product with h, h's own rounding), the three other products 3, exp(-|g|) with its correction 4 (exp2's own ulp, the constant's and the correction's rounding, the
    last fma), 1 + t 1, reciprocal 2, t / (1 + t) 1: 33, wherever g is.  Without the correction -80 alone would take 40 more, and the odds that no sample of 40 000 shows it
    are nil: the sum below is over what a gate near zero (|g| < 1) is off by on the same rows, which holds all but the sigmoid's own part."""
    g = torch.Generator().manual_seed(2)
    h = torch.randn(200, 200, generator=g).to(dev())
    zero, one = torch.zeros_like(h), torch.ones(200, device=dev())

    def off(gate):
        gate = gate.to(dev())
        y = trunk.gated_residual(zero, h, gate, one, None, 1.0, "sigmoid", 0.0).double()
        n = h.double() / torch.sqrt((h.double() ** 2).mean(-1, keepdim=True))
        want = n / (1 + torch.exp(-gate.double()))
        return float(((y - want).abs() / want.abs()).max()) / E
    near, far = off(torch.rand(200, 200, generator=g) * 2 - 1), off(torch.rand(200, 200, generator=g) * 160 - 80)
    assert far <= 33 and far <= near + 8
    bad = torch.tensor([float("inf"), -float("inf"), float("nan"), 3e38, -3e38, 104.0, -104.0, 0.0]).repeat(200, 25).to(dev())
    mine = {"gate": bad.requires_grad_(True), "h": h.clone().requires_grad_(True)}
    y = trunk.gated_residual(zero, mine["h"], mine["gate"], one, None, 1.0, "sigmoid")
    n = trunk.gated_residual(zero, h, None, one, None)
    assert torch.equal(y[:, 0::8], n[:, 0::8]) and torch.equal(y[:, 3::8], n[:, 3::8]) and not y[:, 1::8].any() and not y[:, 4::8].any()
    assert bool(y[:, 2::8].isnan().all()) and int(y.isnan().sum()) == 200 * 25
    dgate, = torch.autograd.grad(y, mine["gate"], torch.where(bad.isnan(), 0.0, 1.0).detach())
    assert not dgate[:, :2].any() and not dgate[:, 3:5].any() and bool(dgate[:, 7].ne(0).all())


def test_refuses_forward_mode_tangents():
    from torch.autograd import forward_ad
    x, w, g = torch.zeros(2, 8), torch.ones(8), torch.zeros(1, 8)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))      # noqa: E731
        for args in ((dual(x), w), (x, dual(w))):
            with pytest.raises(NotImplementedError, match="pre_norm has no forward-mode derivative"):
                trunk.pre_norm(*args)
        whole = (x, x, g, w, w)
        for k in range(5):
            with pytest.raises(NotImplementedError, match="gated_residual has no forward-mode derivative"):
                trunk.gated_residual(*(dual(t) if i == k else t for i, t in enumerate(whole)))


@pytest.mark.gpu
def test_residual_refuses_a_gradient_with_a_tangent():
    from torch.autograd import forward_ad
    x, w = torch.randn(3, 40, device=dev(), requires_grad=True), torch.ones(40, device=dev())
    y, u = trunk.gated_residual(x, x, None, w, w)
    with forward_ad.dual_level():
        for out in (y, u):
            with pytest.raises(NotImplementedError, match="the gradient of gated_residual has no forward-mode derivative"):
                torch.autograd.grad(out, x, forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y)), retain_graph=True)


@pytest.mark.filterwarnings("ignore")
def test_conditioning_operators_refuse_to_be_traced():
    """A tracer would keep the output's allocation and drop the kernel."""
    from torch.fx.experimental.proxy_tensor import make_fx
    x, w, ids, table = torch.zeros(2, 8), torch.ones(8), torch.zeros(2, dtype=torch.int64), torch.zeros(3, 8)
    q, e = torch.zeros(5, 128, dtype=torch.float8_e4m3fn), torch.zeros(1, 1, dtype=torch.uint8)
    for name, f in (("pre_norm", lambda t: trunk.pre_norm(t, w)), ("gated_residual", lambda t: trunk.gated_residual(t, t, None, w)), ("lookup", lambda t: codes.lookup(ids, t)),
                    ("linear8", lambda t: quantize.linear8(t, q, e)), ("quantize_blocks", lambda t: quantize.quantize_blocks(t)[0]),
                    ("dequantize_blocks", lambda t: quantize.dequantize_blocks(q, e, 100, 128) + t.sum())):
        arg = table if name == "lookup" else x
        for record in (lambda: torch.jit.trace(f, arg, check_trace=False), lambda: make_fx(f)(arg), lambda: make_fx(f, tracing_mode="fake")(arg)):
            with pytest.raises(RuntimeError, match=f"{name} cannot be recorded"):
                record()
        with pytest.raises(RuntimeError, match="HIP device"):
            f(arg)


@pytest.mark.gpu
def test_conditioning_operators_traced_gradients_and_compiled_calls():
    from torch.fx.experimental.proxy_tensor import make_fx
    x, w = torch.randn(3, 40, device=dev(), requires_grad=True), torch.ones(40, device=dev())
    table = torch.randn(5, 8, device=dev(), requires_grad=True)
    for out, leaf in ((trunk.pre_norm(x, w), x), (codes.lookup(torch.tensor([1, 2], device=dev()), table), table)):
        with pytest.raises(RuntimeError, match="cannot be recorded"):
            make_fx(lambda d: torch.autograd.grad(out, leaf, d)[0])(torch.ones_like(out))
    f = lambda t: trunk.pre_norm(t, w) * 2      # noqa: E731
    with torch.no_grad():
        assert torch.equal(torch.compile(f, backend="eager")(x), f(x))      # torch.compile leaves the call out of its graphs and makes it as it is


def test_factors_beyond_32_bits_are_refused():
    """The kernels take scale and eps in 32 bits, where these would be infinite."""
    x, w = torch.zeros(2, 8), torch.ones(8)
    for big in (1e39, -1e39, 1.7e308):
        with pytest.raises(RuntimeError, match="scale must be finite"):
            trunk.gated_residual(x, x, None, w, scale=big)
        with pytest.raises(RuntimeError, match="scale must be finite"):
            codes.lookup(torch.zeros(3, dtype=torch.int64), x, scale=big)
        with pytest.raises(RuntimeError, match="eps must be finite"):
            trunk.pre_norm(x, w, eps=abs(big))
    with pytest.raises(RuntimeError, match="HIP device"):
        trunk.gated_residual(x, x, None, w, scale=3e38, eps=3e38)


@pytest.mark.gpu
def test_views_that_negate_are_read_as_they_are():
    """A view with torch's negative bit (the imaginary part of a conjugate) holds the other sign in memory."""
    neg = lambda t: torch._neg_view(t)      # noqa: E731
    x, h, w, ids = torch.randn(5, 24, device=dev()), torch.randn(5, 24, device=dev()), torch.randn(24, device=dev()), torch.tensor([3, 0, 4, 4], device=dev())
    for a, b in zip(trunk.gated_residual(neg(x), neg(h), neg(x), neg(w), neg(w), 0.5, "sigmoid"), trunk.gated_residual(-x, -h, -x, -w, -w, 0.5, "sigmoid")):
        assert torch.equal(a, b)
    assert torch.equal(trunk.pre_norm(neg(x), w), trunk.pre_norm(-x, w))
    assert torch.equal(codes.lookup(ids, neg(x)), -x[ids]) and torch.equal(codes.lookup(neg(-ids), x), x[ids])
    one = torch.complex(x[:, :1], h[:, :1]).conj().imag
    assert one.is_neg() and torch.equal(codes.lookup(ids, one), -h[ids, :1])
    (q, e), (p, f) = quantize.quantize_blocks(neg(x), 1), quantize.quantize_blocks(-x, 1)
    assert torch.equal(q.view(torch.uint8), p.view(torch.uint8)) and torch.equal(e, f)
    q, e = quantize.quantize_blocks(h, 128)
    assert torch.equal(quantize.linear8(neg(x), q, e, neg(x[:, 0].clone())), quantize.linear8(-x, q, e, -x[:, 0]))
    leaf = x.clone().requires_grad_(True)
    got, = torch.autograd.grad(trunk.pre_norm(neg(leaf), w), leaf, neg(h))
    want, = torch.autograd.grad(trunk.pre_norm(-leaf, w), leaf, -h)
    assert torch.equal(got, want)
    table = x.clone().requires_grad_(True)
    got, = torch.autograd.grad(codes.lookup(ids, table), table, neg(h[:4]))
    assert torch.equal(got, torch.autograd.grad(codes.lookup(ids, table), table, -h[:4])[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [B16, F16])
def test_trunk_in_eight_bits_on_16_bit_streams(dtype):
    """to_8bit() and a cast, in either order: the layers' weights are quantised from what the trunk holds at that time."""
    torch.manual_seed(3)
    stack = trunk.Trunk(96, 2).to(dev())
    x = torch.randn(20, 96, device=dev()).to(dtype)
    with torch.no_grad():
        got = stack.to_8bit().to(dtype)(x)
        want = stack.to_8bit()(x.float())
        assert got.dtype == dtype
        # the same 8-bit weights; streams rounded to 16 bits some eight times a block, and activations that then round to another e4m3 number (2^-4) where they lay near a
        # border, a share of about 2^-9 / 2^-4 of them: 2 blocks * (8 * 2^-9 + 3 products * 2^-4 * (2^-5)^0.5) = 0.1 of the latent's size at the most
        assert float((got.float() - want).norm() / want.norm()) <= 0.1
        late = trunk.Trunk(96, 2).to(dev())
        late.load_state_dict(stack.state_dict())
        assert late.to(dtype).to_8bit()(x).dtype == dtype


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,wdtype", TYPES[1:])
@pytest.mark.parametrize("shape,gate", [((4, 6, 32), (4, 1, 32)), ((3, 2, 5, 40), (3, 1, 1, 40)), ((2, 4000, 24), (2, 1, 24)), ((700, 3, 130), (700, 1, 130)), ((2, 1500, 1030), (2, 1, 1030)),
                                        ((1, 900, 4096), (1, 1, 4096)), ((4, 5, 6, 2048), (4, 1, 1, 2048))])
def test_residual_shared_gates_of_16_bits(shape, gate, dtype, wdtype):
    for form, act in (("both", "sigmoid"), ("last", None)):
        leaf, seeds = make(shape, dtype, wdtype, form, gate, sum(shape))
        check(leaf, seeds, -0.5, act)


@pytest.mark.gpu
def test_the_readmes_example_runs():
    import os
    import re
    from nvp_amd import modulation
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "README.md")).read()
    code, = [b for b in re.findall(r"```python\n(.*?)```", text, re.S) if "CodeTable" in b]
    net = modulation.SirenNet(dim_in=1, dim_hidden=128, dim_out=3, num_layers=3, w0_initial=30.)
    ids = torch.randint(-1, 600, (500,), device=dev())
    names = {"torch": torch, "siren_wrapper": modulation.SirenWrapper(net, latent_dim=114).to(dev()), "coords": ids[:, None].float() / 600, "frame_ids": ids}
    exec(code, names)
    assert names["rgb"].shape == (500, 3) and bool(names["rgb"].isfinite().all()) and not names["rgb"].requires_grad
