"""8-bit linear layers (nvp_amd.quantize.linear8 and its block form) against a plain 64-bit evaluation, and their refusals.

Tolerances.  Quantisation is exact to state: the scale is a power of two, v * 2^-s is exact in fp32 unless it falls below the normal numbers
(and then it rounds to an e4m3 zero either way), and e4m3 rounds to nearest even - so block forms are compared for equality.  A product sums K
values that are exact in fp32; each of at most K fp32 additions (plus one for the bias) rounds by at most one step, 2^-23 of a partial sum that
never exceeds S = sum |x||w| + |bias|, and the result is rounded once to its type by at most eps / 2 of itself:
|y - exact| <= (K + 1) 2^-23 S + eps / 2 |exact| (+ the smallest number of the type, for results below its normal numbers).
16-bit streams run on the 8-bit matrix instructions, which drop, inside each group of 8 products, what lies more than 13 bits below the largest
product's exponent: at most 7 * 2^-13 of the group's largest product, so at most 7 * 2^-13 S in all.  That worst case is loose; where signs are
random the dropped parts (uniform below 2^-13 G, G about 3.5 times the products' rms) add up to 2^-13 * 3.5 / sqrt(3) = 2.5e-4 of the result's
norm, which is asserted too, next to eps / 2 for the rounding."""
import ctypes

import pytest
import torch

from nvp_amd import _lib as L
from nvp_amd import quantize as Q

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def dev():
    return torch.device("cuda:0")


def plain_blocks(v, rows):
    """(values the block form stands for, scale exponents) in float64, from the definition; non-finite elements become NaN."""
    v = v.detach().double().cpu()
    r, k = v.shape
    b = torch.nn.functional.pad(v, (0, -k % 128, 0, -r % rows)).reshape(-(-r // rows), rows, -(-k // 128), 128)
    fin = torch.where(torch.isfinite(b), b, torch.zeros_like(b))
    top = fin.abs().amax((1, 3))
    m, x = torch.frexp(top)                                       # 448 = 0.875 * 2^9
    s = torch.where(top > 0, (x - 9 + (m > 0.875)).clamp(min=-127), torch.zeros_like(x))
    up = torch.exp2(s.double())[:, None, :, None]
    t = fin / up
    step = torch.exp2(torch.floor(torch.log2(t.abs().clamp(min=2.0 ** -6))) - 3)
    t = torch.round(t / step) * step * up
    t = torch.where(torch.isfinite(b), t, torch.full_like(t, float("nan")))
    return t.reshape(-1, b.shape[2] * 128)[:r, :k], s


def plain_linear(x, w, bias):
    xq, _ = plain_blocks(x, 1)
    wq, _ = plain_blocks(w, 128)
    y, s = xq @ wq.t(), xq.abs() @ wq.abs().t()
    if bias is not None:
        y, s = y + bias.double().cpu(), s + bias.double().cpu().abs()
    return y, s


def within(got, y, s, k, dtype):
    half = torch.finfo(dtype).eps / 2
    drop = 0.0 if dtype == torch.float32 else 7 * 2.0 ** -13
    tol = ((k + 1) * 2.0 ** -23 + drop) * s * (1 + half) + half * y.abs() + torch.finfo(dtype).tiny
    err = (got.double().cpu() - y).abs()
    assert bool((err <= tol).all()), float((err - tol).max())
    norm = 4e-7 * k ** 0.5 + half if dtype == torch.float32 else 2.5e-4 + half
    if y.numel() >= 1000:
        assert float(err.norm() / y.norm()) <= norm


# ---- on the host ----------------------------------------------------------------------------------------------------------------------------
def test_refusals_on_the_host():
    x, q, e = torch.zeros(3, 200), torch.zeros(5, 256, dtype=torch.float8_e4m3fn), torch.zeros(1, 2, dtype=torch.uint8)
    with pytest.raises(RuntimeError, match="HIP device"):
        Q.linear8(x, q, e)
    with pytest.raises(RuntimeError, match="HIP device"):
        Q.quantize_blocks(x)
    with pytest.raises(RuntimeError, match="HIP device"):
        Q.dequantize_blocks(q, e, 200, rows=128)
    with pytest.raises(RuntimeError, match="columns in blocks"):
        Q.linear8(torch.zeros(3, 300), q, e)                       # three blocks of x, two of the weight
    with pytest.raises(RuntimeError, match="columns in blocks"):
        Q.linear8(x, q, torch.zeros(2, 2, dtype=torch.uint8))
    with pytest.raises(RuntimeError, match="float8_e4m3fn"):
        Q.linear8(x, q.to(torch.float32), e)
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        Q.linear8(x.double(), q, e)
    with pytest.raises(RuntimeError, match="bias must be"):
        Q.linear8(x, q, e, torch.zeros(4))
    with pytest.raises(RuntimeError, match="bias must be"):
        Q.linear8(x, q, e, torch.zeros(5, dtype=torch.bfloat16))
    with pytest.raises(NotImplementedError, match="inference-only"):
        Q.linear8(x.requires_grad_(True), q, e)
    with pytest.raises(RuntimeError, match="no rows"):
        Q.linear8(torch.zeros(3, 200), q[:0], e[:0])
    with pytest.raises(RuntimeError, match="a block has 1 or 128 rows"):
        Q.quantize_blocks(torch.zeros(4, 4), rows=64)
    with pytest.raises(RuntimeError, match="matrix"):
        Q.quantize_blocks(torch.zeros(4))
    with pytest.raises(ValueError):
        Q.Linear8(0, 5)


def test_entry_points_refuse_bad_arguments_without_a_device():
    lib, d = L.load(), ctypes.c_void_p(64)                          # never dereferenced
    assert lib.nvp_linear8_workspace_bytes(2, 4096, 4096) == 0 and lib.nvp_linear8_workspace_bytes(16, 4096, 4096) > 0
    assert lib.nvp_linear8_workspace_bytes(1000, 300, 1130) >= 1000 * 384 + 1000 * 3 + 9 * 3
    assert lib.nvp_linear8_workspace_bytes(-1, 128, 128) == L.ERR_BADARG and lib.nvp_linear8_workspace_bytes(4, 0, 128) == L.ERR_BADARG
    need = lib.nvp_linear8_workspace_bytes(1000, 128, 1128)
    for args in ((None, d, d, d), (d, None, d, d), (d, d, None, d), (d, d, d, None)):
        x, q, e, y = args
        assert lib.nvp_linear8(x, 0, q, e, None, y, 1000, 128, 1128, d, need, None) == L.ERR_BADARG
        assert lib.nvp_linear8(x, 0, q, e, None, y, 0, 128, 1128, d, need, None) == 0
    assert lib.nvp_linear8(d, 3, d, d, None, d, 1000, 128, 1128, d, need, None) == L.ERR_BADARG             # no such type
    assert lib.nvp_linear8(d, 0, ctypes.c_void_p(8), d, None, d, 1000, 128, 1128, d, need, None) == L.ERR_BADARG      # q not 16-byte aligned
    assert lib.nvp_linear8(d, 0, d, d, None, d, 1000, 128, 1128, None, need, None) == L.ERR_BADARG
    assert lib.nvp_linear8(d, 0, d, d, None, d, 1000, 128, 1128, d, need - 1, None) == L.ERR_BADARG
    assert lib.nvp_quantize_blocks(d, 0, d, d, 4, 4, 64, None) == L.ERR_BADARG
    assert lib.nvp_quantize_blocks(None, 0, d, d, 4, 4, 1, None) == L.ERR_BADARG
    assert lib.nvp_dequantize_blocks(d, d, None, 0, 4, 4, 1, None) == L.ERR_BADARG


# ---- on the device --------------------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,rows", [((1, 1), 1), ((3, 127), 1), ((129, 260), 128), ((256, 128), 128), ((5, 1000), 128)])
def test_block_form(shape, rows, dtype):
    g = torch.Generator().manual_seed(shape[0] * 1000 + shape[1])
    v = torch.randn(shape, generator=g) * torch.exp(3 * torch.randn(shape[0], 1, generator=g))
    v[0, 0] = 448.0
    v = v.to(dtype).to(dev())
    q, e = Q.quantize_blocks(v, rows)
    want, s = plain_blocks(v, rows)
    assert q.shape == (shape[0], -(-shape[1] // 128) * 128) and torch.equal(e.cpu().long() - 127, s.long())
    back = Q.dequantize_blocks(q, e, shape[1], rows, torch.float32)
    assert torch.equal(back.cpu().double(), want)
    assert not q.view(torch.uint8)[:, shape[1]:].any()


@pytest.mark.gpu
def test_block_form_at_the_borders():
    """Every e4m3 number and every midpoint between two of them; blocks of zeros, of the smallest and the largest floats; non-finite values."""
    codes = torch.arange(0, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    mid = (codes[1:] + codes[:-1]) / 2
    block = torch.zeros(6, 256)
    block[0, :127], block[0, 128:254] = codes, mid
    block[0, 254] = 448.0
    block[1, :127] = -codes
    block[2, 0] = 2.0 ** -149
    block[3, :2] = torch.tensor([3.4028234e38, -1e38])
    block[4, :3] = torch.tensor([float("inf"), 1.0, float("nan")])
    block[5, 128] = 448.0000305                                    # one step above: the next power
    q, e = Q.quantize_blocks(block.to(dev()), 1)
    want, s = plain_blocks(block, 1)
    assert torch.equal(e.cpu().long() - 127, s.long())
    back = Q.dequantize_blocks(q, e, 256, 1).cpu()
    want = want.float()                          # the largest float rounds up to 2^128, which is infinite in the fp32 that comes back
    assert bool(back[3, 0].isinf()) and int(back.isinf().sum()) == 1
    assert torch.equal(back.nan_to_num(nan=7.0), want.nan_to_num(nan=7.0)) and int(back.isnan().sum()) == 2


SHAPES = [(1, 1, 1), (1, 128, 16), (2, 130, 17), (16, 4096, 100), (17, 256, 128), (33, 129, 300), (64, 1000, 65), (513, 384, 129), (600, 100, 1000), (700, 640, 4099),
          (4099, 300, 2050), (1, 1100, 5003), (8, 8192, 256), (16, 9000, 40), (9, 16000, 2100), (32, 3000, 50), (300, 4000, 70), (400, 200, 6000), (77, 1100, 5003), (200, 9000, 300),
          (2048, 242, 128), (2049, 1, 1), (2100, 127, 61), (3001, 130, 200), (2500, 300, 65), (5000, 128, 256), (2777, 515, 100)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_linear8(m, k, n, dtype):
    g = torch.Generator().manual_seed(m + 7 * k + 13 * n)
    x = (torch.randn(m, k, generator=g) * torch.exp(torch.randn(m, 1, generator=g))).to(dtype)
    w = torch.randn(n, k, generator=g) * k ** -0.5
    bias = torch.randn(n, generator=g).to(dtype) if (m + n) % 2 else None
    q, e = Q.quantize_blocks(w.to(dev()), 128)
    y = Q.linear8(x.to(dev()), q, e, bias.to(dev()) if bias is not None else None)
    assert y.dtype == dtype and y.shape == (m, n)
    want, s = plain_linear(x, w, bias)
    within(y, want, s, k, dtype)


@pytest.mark.gpu
def test_linear8_scales_of_every_block_count():
    """Blocks whose scales lie far apart, in x and in the weight: a scale that is taken from a neighbouring row or block shows at once."""
    g = torch.Generator().manual_seed(3)
    for m, n in ((5, 2100), (40, 2100), (300, 2100), (4100, 2100), (4100, 70), (2100, 40)):
        k = 128 * 5 + 3
        x = torch.randn(m, k, generator=g) * torch.exp2(torch.randint(-12, 13, (m, -(-k // 128)), generator=g).float()).repeat_interleave(128, 1)[:, :k]
        up = torch.exp2(torch.randint(-12, 13, (-(-n // 128), -(-k // 128)), generator=g).float())
        w = torch.randn(n, k, generator=g) * up.repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
        q, e = Q.quantize_blocks(w.to(dev()), 128)
        want, s = plain_linear(x, w, None)
        within(Q.linear8(x.to(dev()), q, e), want, s, k, torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(3, 2060), (100, 2060), (5000, 2060), (5000, 60)])
def test_linear8_rows_with_non_finite_values_are_nan_and_no_others(m, n):
    g = torch.Generator().manual_seed(m)
    x, w = torch.randn(m, 200, generator=g), torch.randn(n, 200, generator=g)
    x[0, 5], x[m - 1, 199] = float("inf"), float("nan")
    q, e = Q.quantize_blocks(w.to(dev()), 128)
    y = Q.linear8(x.to(dev()), q, e).cpu()
    assert bool(y[0].isnan().all()) and bool(y[m - 1].isnan().all()) and bool(y[1:m - 1].isfinite().all())


@pytest.mark.gpu
def test_linear8_empty_strided_and_batched_inputs():
    w = torch.randn(70, 96, device=dev())
    q, e = Q.quantize_blocks(w, 128)
    assert Q.linear8(torch.zeros(0, 96, device=dev()), q, e).shape == (0, 70)
    assert Q.linear8(torch.zeros(2, 0, 96, device=dev()), q, e).shape == (2, 0, 70)
    x = torch.randn(4, 9, 200, device=dev())
    a = Q.linear8(x[..., 3:99], q, e)                               # rows 200 apart, not 16-byte aligned
    b = Q.linear8(x[..., 3:99].contiguous(), q, e)
    c = Q.linear8(x.transpose(0, 1)[..., 3:99], q, e).transpose(0, 1)
    assert a.shape == (4, 9, 70) and torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.gpu
def test_linear8_rows_do_not_depend_on_their_neighbours():
    """The same row gives the same bits alone, in a small batch of its path, and with other rows around it."""
    x, w = torch.randn(5000, 300, device=dev()), torch.randn(2100, 300, device=dev())
    q, e = Q.quantize_blocks(w, 128)
    full = Q.linear8(x, q, e)
    assert torch.equal(full, Q.linear8(x, q, e))
    assert torch.equal(full[:4990], Q.linear8(x[:4990], q, e))
    few = Q.linear8(x[:16], q, e)
    assert torch.equal(few[:3], Q.linear8(x[:3], q, e))


@pytest.mark.gpu
def test_linear8_module_and_its_state():
    lin = torch.nn.Linear(114, 128).to(dev())
    m = Q.Linear8.from_linear(lin)
    x = torch.randn(50, 114, device=dev())
    want, s = plain_linear(x.cpu(), lin.weight, lin.bias)
    within(m(x), want, s, 114, torch.float32)
    other = Q.Linear8(114, 128, device=dev())
    other.load_state_dict(m.state_dict())
    assert torch.equal(other(x), m(x))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 300, 4200])
def test_linear8_captured_and_replayed(m):
    x, w, b = torch.randn(m, 260, device=dev()), torch.randn(2060, 260, device=dev()), torch.randn(2060, device=dev())
    q, e = Q.quantize_blocks(w, 128)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        Q.linear8(x, q, e, b)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = Q.linear8(x, q, e, b)
    for _ in range(3):
        x.copy_(torch.randn(m, 260, device=dev()))
        graph.replay()
        want = Q.linear8(x, q, e, b)
        torch.cuda.synchronize()
        assert torch.equal(y, want)


@pytest.mark.gpu
def test_linear8_two_streams_at_once():
    x, w = torch.randn(2, 3000, 512, device=dev()), torch.randn(1100, 512, device=dev())
    q, e = Q.quantize_blocks(w, 128)
    want = [Q.linear8(x[i], q, e) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got.append((i, Q.linear8(x[i], q, e)))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i, y in got)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", [(20, 300, 8200), (33, 640, 70), (65, 129, 8191), (511, 1300, 4100), (1500, 700, 4100), (4200, 1300, 2300)])
def test_linear8_every_tile(m, k, n, dtype):
    """32 columns a workgroup; 64 x 64 tiles, full and ragged; 128 x 128 with one and with two tiles per CU; 256 x 256 with more blocks than stages."""
    test_linear8(m, k, n, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(40, 500), (511, 4100), (1500, 4100), (20, 8200)])
def test_linear8_captured_tiles(m, n):
    k = 1300
    x, w = torch.randn(m, k, device=dev()), torch.randn(n, k, device=dev())
    q, e = Q.quantize_blocks(w, 128)
    Q.linear8(x, q, e)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = Q.linear8(x, q, e)
    for _ in range(3):
        x.copy_(torch.randn(m, k, device=dev()))
        graph.replay()
        want = Q.linear8(x, q, e)
        torch.cuda.synchronize()
        assert torch.equal(y, want)


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", [(1_100_000, 2048, 300), (9_000_000, 256, 250)])
def test_linear8_offsets_past_32_bits(m, k, n):
    x = torch.randn(m, k, device=dev(), dtype=torch.bfloat16)
    w = torch.randn(n, k) * k ** -0.5
    q, e = Q.quantize_blocks(w.to(dev()), 128)
    y = Q.linear8(x, q, e)
    for a in (0, 2 ** 31 // k - 20, 2 ** 31 // n - 20, m - 40):
        a = min(a, m - 40)
        want, s = plain_linear(x[a:a + 40].cpu(), w, None)
        within(y[a:a + 40], want, s, k, torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", [(8200, 128, 1), (33003, 130, 61), (32769, 129, 64), (66001, 242, 128), (49999, 300, 50), (65601, 128, 250), (33000, 128, 65), (131073, 515, 33)])
def test_linear8_few_columns(m, k, n, dtype):
    test_linear8(m, k, n, dtype)


@pytest.mark.gpu
def test_linear8_few_columns_scales_non_finite_values_and_replays():
    g = torch.Generator().manual_seed(4)
    m, k, n = 50001, 259, 40
    x = torch.randn(m, k, generator=g) * torch.exp2(torch.randint(-12, 13, (m, 3), generator=g).float()).repeat_interleave(128, 1)[:, :k]
    w = torch.randn(n, k, generator=g) * torch.exp2(torch.randint(-12, 13, (1, 3), generator=g).float()).repeat_interleave(128, 1)[:, :k]
    q, e = Q.quantize_blocks(w.to(dev()), 128)
    want, s = plain_linear(x, w, None)
    mine = x.to(dev())
    y = Q.linear8(mine, q, e)
    within(y, want, s, k, torch.float32)
    bad = mine.clone()
    bad[0, 5], bad[m - 1, 258] = float("inf"), float("nan")
    z = Q.linear8(bad, q, e)
    assert bool(z[0].isnan().all()) and bool(z[m - 1].isnan().all()) and torch.equal(z[1:m - 1], y[1:m - 1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = Q.linear8(mine, q, e)
    for _ in range(3):
        mine.copy_(mine.roll(1, 0))
        graph.replay()
        want = Q.linear8(mine, q, e)
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_linear8_refuses_forward_mode_tangents():
    from torch.autograd import forward_ad
    x, q, e, b = torch.zeros(3, 200), torch.zeros(5, 256, dtype=torch.float8_e4m3fn), torch.zeros(1, 2, dtype=torch.uint8), torch.zeros(5)
    with forward_ad.dual_level():
        for args in ((forward_ad.make_dual(x, x.clone()), q, e, None), (x, q, e, forward_ad.make_dual(b, b.clone()))):
            with pytest.raises(NotImplementedError, match="linear8 has no forward-mode derivative"):
                Q.linear8(*args)


@pytest.mark.parametrize("cast", [lambda m: m.half(), lambda m: m.bfloat16(), lambda m: m.double().float(), lambda m: m.to(torch.float16), lambda m: m.to("cpu", torch.bfloat16),
                                  lambda m: m.type(torch.float16), lambda m: m.to("meta"), lambda m: m.to_empty(device="cpu"), lambda m: torch.nn.Sequential(m).half()[0]])
def test_linear8_module_keeps_its_weight_through_casts(cast):
    """Casts concern the bias: the weight's bytes and scales stay what they are, wherever the module is in a tree."""
    m = Q.Linear8(200, 130)
    raw = torch.arange(130 * 256).to(torch.uint8).view(130, 256)
    m.q, m.e, m.bias = raw.view(torch.float8_e4m3fn), torch.tensor([[1, 2], [3, 4]], dtype=torch.uint8), torch.arange(130.0)
    names = list(m.state_dict())
    m = cast(m)
    assert m.q.dtype == torch.float8_e4m3fn and m.e.dtype == torch.uint8 and m.q.shape == (130, 256) and m.e.shape == (2, 2)
    assert m.q.device == m.e.device == m.bias.device and list(m.state_dict()) == names
    if m.q.device.type == "cpu" and not cast.__code__.co_names[0] == "to_empty":
        assert torch.equal(m.q.view(torch.uint8), raw) and m.e.tolist() == [[1, 2], [3, 4]] and torch.equal(m.bias.float(), torch.arange(130.0))
    assert m.bias.dtype != torch.float64
    bare = Q.Linear8(5, 5, bias=False).half()
    assert bare.bias is None and bare.q.dtype == torch.float8_e4m3fn


def test_linear8_module_is_whole_after_a_move_that_fails():
    m = Q.Linear8(200, 130)
    q, e = m.q, m.e

    def fails(t):
        raise ValueError("no")
    with pytest.raises(ValueError):
        m._apply(fails)
    assert m.q is q and m.e is e


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_linear8_module_of_every_stream_type(dtype):
    """An fp32 layer's 8-bit form, cast to the stream's type: the weight in the same bytes, and the call's result that of the operator."""
    torch.manual_seed(1)
    lin = torch.nn.Linear(300, 70).to(dev())
    m = Q.Linear8.from_linear(lin)
    q, e = m.q.clone(), m.e.clone()
    m = m.to(dtype).cpu().to(dev())
    x = torch.randn(40, 300, device=dev()).to(dtype)
    assert torch.equal(m.q.view(torch.uint8), q.view(torch.uint8)) and torch.equal(m.e, e)
    y = m(x)
    assert y.dtype == dtype and torch.equal(y, Q.linear8(x, q, e, lin.bias.detach().to(dtype)))
    want, s = plain_linear(x.cpu(), lin.weight, lin.bias.detach().to(dtype))
    within(y, want, s, 300, dtype)


def other_layouts(q, e):
    """The block form (q, e) in other places: a slice of wider rows, a contiguous matrix at an odd address, a transposed one; scales transposed."""
    raw = q.view(torch.uint8)
    r, k = raw.shape
    wide = torch.zeros(r, k + 600, device=q.device, dtype=torch.uint8)
    wide[:, 3:3 + k] = raw
    odd = torch.zeros(r * k + 1, device=q.device, dtype=torch.uint8)[1:].view(r, k)
    odd.copy_(raw)
    turned, scales = raw.t().contiguous().t(), e.t().contiguous().t()
    assert odd.is_contiguous() and odd.data_ptr() % 16 == 1 and not turned.is_contiguous() and not scales.is_contiguous()
    return [(t.view(torch.float8_e4m3fn), scales) for t in (wide[:, 3:3 + k], odd, turned)]


@pytest.mark.gpu
def test_dequantize_blocks_of_any_stride_and_alignment():
    q, e = Q.quantize_blocks(torch.randn(140, 300, device=dev()), 128)
    want = Q.dequantize_blocks(q, e, 300, 128)
    assert all(torch.equal(Q.dequantize_blocks(p, f, 300, 128), want) for p, f in other_layouts(q, e))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [3, 100, 5000])
def test_linear8_weights_of_any_stride_and_alignment(m):
    x = torch.randn(m, 300, device=dev())
    q, e = Q.quantize_blocks(torch.randn(140, 300, device=dev()), 128)
    want = Q.linear8(x, q, e)
    assert all(torch.equal(Q.linear8(x, p, f), want) for p, f in other_layouts(q, e))


@pytest.mark.gpu
def test_block_form_of_more_blocks_and_values_than_one_launch_takes():
    """2^24 blocks of a row each (2^32 threads) and more than 2^32 values: the parts on both sides of a launch's end, and the last rows, as the same rows alone."""
    rows, k = (1 << 24) + 77, 260                                   # three blocks a row; 4.36e9 values
    v = torch.randn(rows, k, device=dev(), dtype=torch.bfloat16)
    spots = [0, (1 << 24) // 3 - 20, (1 << 25) // 3 - 20, (1 << 32) // k - 20, (1 << 24) - 20, rows - 40]
    q, e = Q.quantize_blocks(v, 1)
    back = Q.dequantize_blocks(q, e, k, 1, torch.bfloat16)
    for a in spots:
        p, f = Q.quantize_blocks(v[a:a + 40], 1)
        assert torch.equal(q[a:a + 40].view(torch.uint8), p.view(torch.uint8)) and torch.equal(e[a:a + 40], f), a
        assert torch.equal(back[a:a + 40], Q.dequantize_blocks(p, f, k, 1, torch.bfloat16)), a
    del q, e, back
    q, e = Q.quantize_blocks(v, 128)
    back = Q.dequantize_blocks(q, e, k, 128, torch.bfloat16)
    for a in spots:
        a = a // 128 * 128
        p, f = Q.quantize_blocks(v[a:a + 256], 128)
        n = p.shape[0]
        assert torch.equal(q[a:a + n].view(torch.uint8), p.view(torch.uint8)) and torch.equal(e[a // 128:a // 128 + f.shape[0]], f), a
        assert torch.equal(back[a:a + n], Q.dequantize_blocks(p, f, k, 128, torch.bfloat16)), a
    del v, q, e, back
    torch.cuda.empty_cache()


@pytest.mark.gpu
def test_linear8_of_more_blocks_than_one_launch_quantises():
    """2^21 rows of 128 blocks and some more: 16 lanes a block are 2^32 threads.  The rows on both sides of the first launch's end as they come out alone."""
    rows, k, n = (1 << 21) + 300, 16384, 20
    if torch.cuda.mem_get_info()[0] < 130 << 30:
        pytest.skip("needs 110 GiB of device memory")
    x = torch.empty(rows, k, device=dev(), dtype=torch.bfloat16)
    x.view(torch.int32)[:] = 0x3f80bf80                             # -1 and 1 in turn
    q, e = Q.quantize_blocks(torch.randn(n, k, device=dev()), 128)
    for a in ((1 << 21) - 80, rows - 100):
        x[a:a + 80] = torch.randn(80, k, device=dev()).to(torch.bfloat16)
    y = Q.linear8(x, q, e)
    for a in (0, (1 << 21) - 100, (1 << 21) - 20, rows - 100):
        # another tile: the same products, in another order: either is within the tolerance above of the exact sum; e4m3 makes |x| larger by 2^-4 at most
        alone = Q.linear8(x[a:a + 100], q, e)
        s = (1 + 2.0 ** -4) * x[a:a + 100].abs().double() @ Q.dequantize_blocks(q, e, k, 128).abs().double().t()
        err = (y[a:a + 100].double() - alone.double()).abs()
        assert bool((err <= 2 * ((k + 1) * 2.0 ** -23 + 7 * 2.0 ** -13) * (1 + 2.0 ** -8) * s + 2 * 2.0 ** -8 * (1 + 2.0 ** -7) * alone.double().abs()).all()), a
        assert float(err.norm() / alone.double().norm()) <= 2 * (2.5e-4 + 2.0 ** -8)
    del x, y
    torch.cuda.empty_cache()


# rows and columns of every path: few rows (x quantised in the workgroup), up to 32 rows, the four tiles, few columns
PATHS = [(2, 2100), (20, 2100), (40, 500), (511, 4100), (1500, 4100), (4100, 2100), (50001, 40), (20000, 130)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["outliers", "log-normal"])
@pytest.mark.parametrize("m,n", PATHS)
def test_linear8_channels_of_very_different_size(m, n, kind, dtype):
    """Some channels of x 30 times the others, or sizes spread over e^6: the small products beside a large one in a group of 8 are what the 8-bit instruction drops.  The
    tolerance holds whatever the sizes: the dropped parts are below 2^-13 G each, at most seven beside the group's largest product G, so their rms is at most
    (7 / 3)^0.5 2^-13 = 1.9e-4 of G, and with random signs the result's is G's at least."""
    g = torch.Generator().manual_seed(m + n)
    k = 643
    size = torch.where(torch.rand(k, generator=g) < 0.05, 30.0, 1.0) if kind == "outliers" else torch.exp(torch.randn(k, generator=g).clamp(-3, 3))
    x = (torch.randn(m, k, generator=g) * size).to(dtype)
    w = torch.randn(n, k, generator=g) * k ** -0.5
    q, e = Q.quantize_blocks(w.to(dev()), 128)
    want, s = plain_linear(x, w, None)
    within(Q.linear8(x.to(dev()), q, e), want, s, k, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES[1:])
@pytest.mark.parametrize("m,n", PATHS)
def test_linear8_scales_far_apart_on_16_bit_streams(m, n, dtype):
    """16-bit streams hand the scale bytes to the matrix instruction: blocks of x and of the weight whose scales lie far apart (as far as fp16 results allow)."""
    g = torch.Generator().manual_seed(m)
    k, (a, b) = 128 * 5 + 3, (12, 12) if dtype == torch.bfloat16 else (5, 3)
    x = torch.randn(m, k, generator=g) * torch.exp2(torch.randint(-a, a + 1, (m, -(-k // 128)), generator=g).float()).repeat_interleave(128, 1)[:, :k]
    up = torch.exp2(torch.randint(-b, b + 1, (-(-n // 128), -(-k // 128)), generator=g).float())
    w = torch.randn(n, k, generator=g) * up.repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    x = x.to(dtype)
    q, e = Q.quantize_blocks(w.to(dev()), 128)
    want, s = plain_linear(x, w, None)
    within(Q.linear8(x.to(dev()), q, e), want, s, k, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES[1:])
@pytest.mark.parametrize("m,n", PATHS)
def test_linear8_non_finite_rows_on_16_bit_streams(m, n, dtype):
    """Rows with an infinity or a NaN, the first and the last, become rows of NaN; every other row keeps its bits.  A weight row with a NaN makes its column NaN."""
    g = torch.Generator().manual_seed(m)
    x, w = torch.randn(m, 643, generator=g).to(dtype).to(dev()), torch.randn(n, 643, generator=g).to(dev())
    q, e = Q.quantize_blocks(w, 128)
    y = Q.linear8(x, q, e)
    bad = x.clone()
    bad[0, 5], bad[m - 1, 642] = float("inf"), float("nan")
    z = Q.linear8(bad, q, e)
    assert bool(z[0].isnan().all()) and bool(z[m - 1].isnan().all()) and torch.equal(z[1:m - 1], y[1:m - 1])
    w[n - 1, 300] = float("nan")
    z = Q.linear8(x, *Q.quantize_blocks(w, 128))
    assert bool(z[:, n - 1].isnan().all()) and bool(z[:, :n - 1].isfinite().all())
