"""Cases of the conditioning operators: learned codes looked up by number, the gated residual step with the norms on both sides of a block,
and the 8-bit linear layer with one power-of-two scale per block of 128.

    lookup      out[i] = scale * table[ids[i]] (a negative id is an empty slot: a row of zeros); gradient: table rows summed over equal ids
    residual    y = x + scale * act(gate) * (h / rms(h)) * post,  u = (y / rms(y)) * next; rms(v)^2 = mean(v^2) + eps; act is the
                identity or the sigmoid; the first norm of a stack has no h, its last step no u
    linear8     y = q(x) q(w)^T + bias with q(v) = e4m3(v / 2^s) * 2^s, one s per row and 128 columns of x, one per 128 x 128 of w;
                s is the smallest power that brings the block's largest value to 448 or below

`own` is set by whoever measures: False computes the plain forms below, True calls the framework."""
import math

import torch

own = False

EPS = 1e-6
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}


def listed():
    return [
        # a training batch of pixels (1 245 184 samples of a 600-frame clip) reads the code of its frame: 32 features, as one keyframe plane gives
        dict(name="lookup frames train", op="lookup", rows=1245184, codes=600, dim=32, dtype="fp32", out="fp32", scale=1.0, skew=0.0, empty=0.0, train=True),
        # a handful of frames asked for by number, odd width (the latent's 114)
        dict(name="lookup few", op="lookup", rows=7, codes=300, dim=114, dtype="fp32", out="fp32", scale=1.0, skew=0.0, empty=0.0, train=False),
        # tokens of a text-like vocabulary, a few of them very frequent, some slots empty; the table stays in 32 bits, the stream is bf16
        dict(name="lookup tokens train", op="lookup", rows=16384, codes=65536, dim=1024, dtype="fp32", out="bf16", scale=32.0, skew=3.0, empty=0.03, train=True),
        # a wide bf16 table and a long ragged batch
        dict(name="lookup long train", op="lookup", rows=200003, codes=50000, dim=512, dtype="bf16", out="bf16", scale=22.62741699796952, skew=2.0, empty=0.0, train=True),
        # one token at a time: latency
        dict(name="residual one row", op="residual", rows=1, dim=4096, dtype="bf16", weights="bf16", gate="row", share=1, act="sigmoid", form="both", scale=0.5, train=False),
        # the modulator's width for config_nvp_l (228) in 32 bits, a gate per row, odd number of rows
        dict(name="residual odd train", op="residual", rows=10007, dim=228, dtype="fp32", weights="fp32", gate="row", share=1, act="none", form="both", scale=1.0, train=True),
        # training: 8 sequences of 2048 with one gate vector each
        dict(name="residual train", op="residual", rows=16384, dim=2048, dtype="bf16", weights="fp32", gate="shared", share=2048, act="sigmoid", form="both", scale=0.25, train=True),
        # a long prompt going through one step of a wide stack
        dict(name="residual long", op="residual", rows=65536, dim=4096, dtype="bf16", weights="bf16", gate="row", share=1, act="sigmoid", form="both", scale=0.5, train=False),
        # one token through a layer: the weights have to be read once
        dict(name="linear8 one row", op="linear8", rows=1, k=4096, n=4096, dtype="bf16", bias=False),
        # a short ragged batch, no size a multiple of the block
        dict(name="linear8 ragged", op="linear8", rows=77, k=1100, n=5003, dtype="fp16", bias=True),
        # a training-size batch of pixels through a modulator layer (128 + 114 inputs, 128 outputs), 32-bit streams
        dict(name="linear8 pixels", op="linear8", rows=1245184, k=242, n=128, dtype="fp32", bias=True),
        # a large product
        dict(name="linear8 large", op="linear8", rows=8192, k=8192, n=8192, dtype="bf16", bias=False),
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], evenly spread over its logarithm."""
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def _width(rng, lo, hi):
    """As _log, half of the time a multiple of 8 and half of the time any number."""
    v = _log(rng, lo, hi)
    return max(8, v // 8 * 8) if rng.random() < 0.5 else v


def draw(rng):
    op = rng.choice(("lookup", "residual", "linear8"))
    if op == "lookup":
        dim = _width(rng, 1, 2048)
        rows, codes = _log(rng, 1, min(1245184, (1 << 27) // dim)), _log(rng, 1, min(200000, (1 << 27) // dim))
        dtype = rng.choice(("fp32", "bf16", "fp16"))
        return dict(op=op, rows=rows, codes=codes, dim=dim, dtype=dtype, out=rng.choice(("fp32", "bf16", "fp16")) if dtype == "fp32" else dtype,
                    scale=rng.choice((1.0, math.sqrt(dim))), skew=rng.choice((0.0, 1.0, 3.0)), empty=rng.choice((0.0, 0.1)), train=rng.random() < 0.6)
    if op == "residual":
        train = rng.random() < 0.5
        dim = _width(rng, 32, 8192)                                                           # rows of a few values: the norm's gradient is a difference of nearly equal numbers
        rows = _log(rng, 1, min(262144, (1 << (25 if train else 27)) // dim))
        gate = rng.choice(("none", "row", "shared"))
        share = 1
        if gate == "shared":
            share = _log(rng, 1, rows)
            rows = rows // share * share
        dtype = rng.choice(("fp32", "bf16", "fp16"))
        return dict(op=op, rows=rows, dim=dim, dtype=dtype, weights=rng.choice(("fp32", dtype)), gate=gate, share=share, act=rng.choice(("none", "sigmoid")),
                    form=rng.choice(("both", "both", "first", "last")), scale=rng.choice((1.0, 0.25)), train=train)
    k, n = _width(rng, 1, 8192), _width(rng, 1, 8192)
    rows = _log(rng, 1, min(1245184, 8192 ** 3 // (k * n), (1 << 28) // (k + n)))
    return dict(op=op, rows=rows, k=k, n=n, dtype=rng.choice(("fp32", "bf16", "fp16")), bias=rng.random() < 0.5)


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(int(seed))

    def normal(*shape, dtype=torch.float32, std=1.0, mean=0.0):
        return (torch.randn(shape, generator=g, device=dev) * std + mean).to(dtype)

    s = {"case": case}
    if case["op"] == "lookup":
        rows, codes, dim = case["rows"], case["codes"], case["dim"]
        r = torch.rand(rows, generator=g, device=dev, dtype=torch.float64)
        ids = (codes * r ** (1.0 + 2.0 * case["skew"])).long().clamp_(max=codes - 1)         # skew > 0: low numbers are frequent
        ids = torch.randperm(codes, generator=g, device=dev)[ids]
        if case["empty"]:
            ids = torch.where(torch.rand(rows, generator=g, device=dev) < case["empty"], torch.full_like(ids, -1), ids)
        s["ids"] = ids
        s["table"] = normal(codes, dim, dtype=TYPES[case["dtype"]], std=dim ** -0.5).requires_grad_(case["train"])
        if case["train"]:
            s["dout"] = normal(rows, dim, dtype=TYPES[case["out"]])
        return s
    if case["op"] == "residual":
        rows, dim, t, w = case["rows"], case["dim"], TYPES[case["dtype"]], TYPES[case["weights"]]
        post, nxt = case["form"] != "first", case["form"] != "last"
        s["x"] = normal(rows, dim, dtype=t, std=1.5)
        if post:
            s["h"] = normal(rows, dim, dtype=t, std=0.7)
            s["post"] = normal(dim, dtype=w, std=0.1, mean=1.0)
            if case["gate"] != "none":
                s["gate"] = normal(rows // case["share"], dim, dtype=t)
        if nxt:
            s["next"] = normal(dim, dtype=w, std=0.1, mean=1.0)
        if case["train"]:
            for k in ("x", "h", "post", "gate", "next"):
                if k in s:
                    s[k].requires_grad_(True)
            if post:
                s["dy"] = normal(rows, dim, dtype=t)
            if nxt:
                s["du"] = normal(rows, dim, dtype=t)
        return s
    rows, k, n, t = case["rows"], case["k"], case["n"], TYPES[case["dtype"]]
    s["x"] = (torch.randn(rows, k, generator=g, device=dev) * torch.exp(torch.randn(rows, 1, generator=g, device=dev))).to(t)
    w = normal(n, k, std=k ** -0.5)
    s["q"], s["e"] = _blocks(w, 128)                                                        # a user's program keeps the layer's weights in this form
    if case["bias"]:
        s["bias"] = normal(n, dtype=t)
    return s


def _power(amax):
    """The smallest whole s with amax <= 448 * 2^s, in [-127, 127]; 0 for a block of zeros."""
    m, x = torch.frexp(amax)                                                                # amax = m * 2^x, 0.5 <= m < 1; 448 = 0.875 * 2^9
    s = x - 9 + (m > 0.875).to(x.dtype)
    return torch.where(amax > 0, s.clamp(-127, 127), torch.zeros_like(s))


def _padded(v, rows):
    """[R, K] -> [ceil(R / rows), rows, ceil(K / 128), 128] with zeros behind the last row and column."""
    r, k = v.shape
    v = torch.nn.functional.pad(v, (0, -k % 128, 0, -r % rows))
    return v.reshape(v.shape[0] // rows, rows, v.shape[1] // 128, 128)


def _blocks(v, rows):
    """32-bit [R, K] -> (e4m3 [R, K rounded up to 128], zeros behind column K; bytes s + 127 [ceil(R / rows), ceil(K / 128)])."""
    b = _padded(v, rows)
    s = _power(b.abs().amax((1, 3)))
    q = (b * torch.exp2(-s.to(torch.float64)).to(torch.float32)[:, None, :, None]).to(torch.float8_e4m3fn)
    return q.reshape(-1, b.shape[2] * 128)[: v.shape[0]].contiguous(), (s + 127).to(torch.uint8)


def run(s):
    c = s["case"]
    return {"lookup": _lookup, "residual": _residual, "linear8": _linear8}[c["op"]](c, s)


def _lookup(c, s):
    if own:
        from nvp_amd import codes
        out = codes.lookup(s["ids"], s["table"], scale=c["scale"], dtype=TYPES[c["out"]])
        if not c["train"]:
            return [out]
        return [out.detach(), torch.autograd.grad(out, s["table"], s["dout"])[0]]
    with torch.no_grad():
        keep = s["ids"] >= 0
        at = s["ids"].clamp(min=0)
        out = (s["table"][at].float() * c["scale"] * keep[:, None]).to(TYPES[c["out"]])
        if not c["train"]:
            return [out]
        d = torch.zeros(s["table"].shape, device=out.device, dtype=torch.float32)
        d.index_add_(0, at, s["dout"].float() * keep[:, None])
        return [out, (d * c["scale"]).to(s["table"].dtype)]


def _residual(c, s):
    if own:
        from nvp_amd import trunk
        act = None if c["act"] == "none" else c["act"]
        if c["form"] == "first":
            outs, seeds = [trunk.pre_norm(s["x"], s["next"], eps=EPS)], [s.get("du")]
        else:
            x, h, gate = s["x"], s["h"], s.get("gate")
            if c["gate"] == "shared":                                                        # [sequences, positions, dim] with a gate [sequences, 1, dim]
                x, h, gate = x.view(-1, c["share"], c["dim"]), h.view(-1, c["share"], c["dim"]), gate.view(-1, 1, c["dim"])
            r = trunk.gated_residual(x, h, gate, s["post"], s.get("next"), scale=c["scale"], gate_act=act, eps=EPS)
            outs, seeds = ([r], [s.get("dy")]) if c["form"] == "last" else (list(r), [s.get("dy"), s.get("du")])
            outs = [o.view(c["rows"], c["dim"]) for o in outs]
        if not c["train"]:
            return outs
        leaves = [s[k] for k in ("x", "h", "gate", "post", "next") if k in s]
        return [o.detach() for o in outs] + list(torch.autograd.grad(outs, leaves, seeds))
    with torch.no_grad():
        t = s["x"].dtype
        x = s["x"].float()
        y, outs = x, []
        if "h" in s:
            h, post = s["h"].float(), s["post"].float()
            r = torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS)
            n = h * r
            gate = s["gate"].float().repeat_interleave(c["share"], 0) if "gate" in s else torch.ones((1, 1), device=x.device)
            a = 1 / (1 + torch.exp(-gate)) if c["act"] == "sigmoid" and "gate" in s else gate
            y = x + c["scale"] * a * n * post
            outs.append(y.to(t))
        if "next" in s:
            nxt = s["next"].float()
            r2 = torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS)
            v = y * r2
            outs.append((v * nxt).to(t))
        if not c["train"]:
            return outs
        d = s["dy"].float() if "h" in s else torch.zeros_like(x)
        dnext = None
        if "next" in s:
            du = s["du"].float()
            dnext = (du * v).sum(0).to(s["next"].dtype)
            dv = du * nxt
            d = d + r2 * (dv - v * (dv * v).mean(-1, keepdim=True))
        grads = [d.to(t)]
        if "h" in s:
            dn = c["scale"] * a * post * d
            grads.append((r * (dn - n * (dn * n).mean(-1, keepdim=True))).to(t))
            if "gate" in s:
                da = c["scale"] * d * n * post
                da = da * a * (1 - a) if c["act"] == "sigmoid" else da
                grads.append(da.reshape(-1, c["share"], c["dim"]).sum(1).to(t))
            grads.append((c["scale"] * a * d * n).sum(0).to(s["post"].dtype))
        return outs + grads + ([dnext] if dnext is not None else [])


def _linear8(c, s):
    if own:
        from nvp_amd import quantize
        return [quantize.linear8(s["x"], s["q"], s["e"], s.get("bias"))]
    k, n = c["k"], c["n"]
    qx, ex = _blocks(s["x"].float(), 1)
    up = lambda e: torch.exp2(e.to(torch.float32) - 127)  # noqa: E731
    x = qx.float() * up(ex).repeat_interleave(128, 1)
    w = s["q"].float() * up(s["e"]).repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)
    y = x @ w.t()
    if "bias" in s:
        y = y + s["bias"].float()
    return [y.to(s["x"].dtype)]


def work(c):
    if c["op"] == "lookup":
        rows, codes, dim, a, b = c["rows"], c["codes"], c["dim"], SIZE[c["dtype"]], SIZE[c["out"]]
        used = codes * (1 - (1 - 1 / codes) ** rows) if not c["skew"] else min(codes, rows)   # table rows that are read at all
        read = min(used, codes) * dim * a + rows * 8
        n = read + rows * dim * b
        return {"bytes": n + (rows * dim * b + codes * dim * a if c["train"] else 0), "flops": rows * dim * (2 if c["train"] else 1)}
    if c["op"] == "residual":
        rows, dim, t, w = c["rows"], c["dim"], SIZE[c["dtype"]], SIZE[c["weights"]]
        post, nxt = c["form"] != "first", c["form"] != "last"
        gate = 0 if not post or c["gate"] == "none" else rows // c["share"]
        streams = 1 + 2 * post + nxt                                                         # x, h, y, u
        n = (streams * rows + gate) * dim * t + (post + nxt) * dim * w
        if c["train"]:                                                                       # dy, du, dx, dh and the gate's and the weights' gradients
            n += ((1 + 2 * post + nxt) * rows + gate) * dim * t + (post + nxt) * dim * w
        return {"bytes": n, "flops": rows * dim * (10 + (30 if c["train"] else 0))}
    rows, k, n, t = c["rows"], c["k"], c["n"], SIZE[c["dtype"]]
    return {"bytes": rows * (k + n) * t + n * k + (n * t if c["bias"] else 0), "flops": 2 * rows * k * n}


def exact(case, seed):
    """The definitions in 64 bits; gradients by differentiating the definition."""
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] == "lookup":
        ids = s["ids"]
        live = torch.nonzero(ids >= 0).flatten()
        out = torch.zeros((c["rows"], c["dim"]), dtype=torch.float64, device=ids.device)
        out[live] = s["table"].detach()[ids[live]].double() * c["scale"]
        if not c["train"]:
            return [out]
        order = torch.argsort(ids[live], stable=True)                                        # equal ids side by side, then differences of running sums would lose digits:
        d = torch.zeros((c["codes"], c["dim"]), dtype=torch.float64, device=ids.device)       # 64-bit adds per row instead
        d.index_add_(0, ids[live][order], s["dout"][live][order].double() * c["scale"])
        return [out, d]
    if c["op"] == "residual":
        leaf = {k: s[k].detach().double().requires_grad_(c["train"]) for k in ("x", "h", "gate", "post", "next") if k in s}
        rms = lambda v: torch.sqrt(torch.mean(v ** 2, -1, keepdim=True) + EPS)  # noqa: E731
        outs, y = [], leaf["x"]
        if "h" in leaf:
            add = leaf["h"] / rms(leaf["h"]) * leaf["post"] * c["scale"]
            if "gate" in leaf:
                gate = torch.sigmoid(leaf["gate"]) if c["act"] == "sigmoid" else leaf["gate"]
                add = (add.reshape(gate.shape[0], -1, c["dim"]) * gate[:, None]).reshape(add.shape)
            y = y + add
            outs.append(y)
        if "next" in leaf:
            outs.append(y / rms(y) * leaf["next"])
        if not c["train"]:
            return outs
        seeds = [s[k].double() for k in ("dy", "du") if k in s]
        return [o.detach() for o in outs] + list(torch.autograd.grad(outs, list(leaf.values()), seeds))
    n, k = c["n"], c["k"]
    x = s["x"].double()
    b = torch.nn.functional.pad(x, (0, -k % 128)).reshape(c["rows"], -1, 128)
    top = b.abs().amax(-1, keepdim=True)
    p = torch.ceil(torch.log2(top / 448))
    p = torch.where(torch.exp2(p - 1) * 448 >= top, p - 1, p)                                 # log2 may round across a whole number
    p = torch.where(torch.exp2(p) * 448 < top, p + 1, p)
    p = torch.where(top > 0, p.clamp(-127, 127), torch.zeros_like(p))
    b = b / torch.exp2(p)
    step = torch.exp2(torch.floor(torch.log2(b.abs().clamp(min=2.0 ** -6))) - 3)              # spacing of e4m3 at this size: 3 bits behind the point, 2^-9 below 2^-6
    xq = (torch.round(b / step) * step * torch.exp2(p)).reshape(c["rows"], -1)
    wq = s["q"].double() * torch.exp2(s["e"].double() - 127).repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)
    y = xq @ wq.t()
    return [y + s["bias"].double() if "bias" in s else y]
