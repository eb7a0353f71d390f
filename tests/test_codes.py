"""Learned codes by number (nvp_amd.codes) against a plain 64-bit evaluation, and their refusals.

Tolerances.  Forward: one fp32 product (2^-24 of it) and one rounding to the output type (eps / 2); exact where scale is 1.  Gradient of a row that c
positions point to: c - 1 fp32 additions and one product, each off by at most 2^-24 of a partial sum that never exceeds S = |scale| sum |dout|, then one
rounding: |got - exact| <= (c + 1) 2^-24 S + eps / 2 |exact| (+ the smallest number of the type)."""
import ctypes

import pytest
import torch

from nvp_amd import _lib as L
from nvp_amd import codes

F32, B16, F16 = torch.float32, torch.bfloat16, torch.float16
E = 2.0 ** -24
PAIRS = [(F32, F32), (F32, B16), (F32, F16), (B16, B16), (F16, F16)]


def dev():
    return torch.device("cuda:0")


def plain(ids, table, scale):
    ids = ids.cpu().long()
    out = table.detach().cpu().double()[ids.clamp(0, table.shape[0] - 1)] * scale
    out[ids < 0] = 0.0
    out[ids >= table.shape[0]] = float("nan")
    return out


def plain_grad(ids, dout, n_codes, scale):
    """(gradient, S, positions per row) in float64"""
    ids, d = ids.cpu().long().flatten(), dout.cpu().double().reshape(-1, dout.shape[-1]) * scale
    ok = (ids >= 0) & (ids < n_codes)
    g, s = torch.zeros(n_codes, d.shape[1], dtype=torch.float64), torch.zeros(n_codes, d.shape[1], dtype=torch.float64)
    g.index_add_(0, ids[ok], d[ok])
    s.index_add_(0, ids[ok], d[ok].abs())
    return g, s, torch.bincount(ids[ok], minlength=n_codes)[:, None].double()


def check(ids, table, scale, dtype):
    t = table.clone().requires_grad_(True)
    out = codes.lookup(ids, t, scale, dtype)
    dtype = table.dtype if dtype is None else dtype
    assert out.dtype == dtype and out.shape == ids.shape + (table.shape[1],)
    want = plain(ids, table, scale)
    half = torch.finfo(dtype).eps / 2
    got = out.detach().double().cpu()
    nan = want.isnan()
    assert torch.equal(got.isnan(), nan)
    err = (got - want).abs()[~nan]
    assert bool((err <= (half + 2.0 ** -24 * (1 + half)) * want.abs()[~nan] + torch.finfo(dtype).tiny).all())
    if scale == 1.0:
        assert torch.equal(got[~nan], want.to(dtype).double()[~nan])
    dout = torch.randn(out.shape, device=out.device).to(dtype)
    g, = torch.autograd.grad(out, t, dout)
    assert g.dtype == table.dtype and g.shape == table.shape
    want, s, c = plain_grad(ids, dout, table.shape[0], scale)
    gh = torch.finfo(table.dtype).eps / 2
    err = (g.double().cpu() - want).abs()
    assert bool((err <= (c + 1) * 2.0 ** -24 * s * (1 + gh) + gh * want.abs() + torch.finfo(table.dtype).tiny).all()), float(err.max())
    assert not g.cpu()[(c == 0).flatten()].any()
    again, = torch.autograd.grad(codes.lookup(ids, t, scale, dtype), t, dout)
    assert torch.equal(g, again)
    return g


# ---- on the host -------------------------------------------------------------------------------------------------------------------------------
def test_refusals_on_the_host():
    ids, table = torch.zeros(3, dtype=torch.int64), torch.zeros(4, 5)
    with pytest.raises(RuntimeError, match="HIP device"):
        codes.lookup(ids, table)
    with pytest.raises(RuntimeError, match="int64 or int32"):
        codes.lookup(ids.float(), table)
    with pytest.raises(RuntimeError, match="int64 or int32"):
        codes.lookup(ids.bool(), table)
    for bad in (torch.zeros(5), torch.zeros(0, 5), torch.zeros(5, 0)):
        with pytest.raises(RuntimeError, match="at least one code"):
            codes.lookup(ids, bad)
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        codes.lookup(ids, table.double())
    with pytest.raises(RuntimeError, match="cannot be read as"):
        codes.lookup(ids, table.bfloat16(), dtype=torch.float32)
    with pytest.raises(RuntimeError, match="cannot be read as"):
        codes.lookup(ids, table, dtype=torch.float64)
    with pytest.raises(RuntimeError, match="finite"):
        codes.lookup(ids, table, scale=float("nan"))
    with pytest.raises(ValueError):
        codes.CodeTable(0, 4)
    m = codes.CodeTable(6, 3, scale=2.0)
    assert list(m.state_dict()) == ["codes"] and m.codes.shape == (6, 3) and float(m.codes.abs().max()) <= 1e-4


def test_entry_points_refuse_bad_arguments_without_a_device():
    lib, d = L.load(), ctypes.c_void_p(64)                             # never dereferenced
    assert lib.nvp_lookup_fwd(None, 1, d, 0, d, 0, 5, 4, 3, 1.0, None) == L.ERR_BADARG
    assert lib.nvp_lookup_fwd(d, 1, d, 1, d, 0, 5, 4, 3, 1.0, None) == L.ERR_BADARG           # a bf16 table read as fp32
    assert lib.nvp_lookup_fwd(d, 1, d, 0, d, 0, 5, 0, 3, 1.0, None) == L.ERR_BADARG
    assert lib.nvp_lookup_fwd(d, 1, d, 0, d, 0, 1 << 31, 4, 3, 1.0, None) == L.ERR_UNSUPPORTED
    assert lib.nvp_lookup_fwd(None, 1, None, 0, None, 0, 0, 4, 3, 1.0, None) == 0
    need = lib.nvp_lookup_bwd_workspace_bytes(5000, 70, 16)
    assert need > 0
    assert lib.nvp_lookup_bwd(d, 1, d, 0, d, 0, 5000, 70, 16, 1.0, d, need - 1, None) == L.ERR_BADARG
    assert lib.nvp_lookup_bwd(d, 1, d, 0, None, 0, 5000, 70, 16, 1.0, d, need, None) == L.ERR_BADARG
    assert lib.nvp_lookup_bwd(d, 1, d, 0, d, 0, 5000, 70, 16, 1.0, ctypes.c_void_p(8), need, None) == L.ERR_BADARG
    assert lib.nvp_lookup_bwd_workspace_bytes(-1, 70, 16) == L.ERR_BADARG


# ---- on the device -----------------------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("table_dtype,dtype", PAIRS)
@pytest.mark.parametrize("n,n_codes,dim", [(1, 1, 1), (3, 2, 7), (50, 1000, 64), (1000, 13, 33), (4096, 600, 32), (4097, 1500, 114), (20000, 5, 1024), (70000, 300, 40), (40000, 70000, 24)])
def test_lookup(n, n_codes, dim, table_dtype, dtype):
    g = torch.Generator().manual_seed(n + n_codes + dim)
    table = torch.randn(n_codes, dim, generator=g).to(table_dtype).to(dev())
    ids = torch.randint(0, n_codes, (n,), generator=g).to(dev())
    check(ids, table, 1.0 if n % 2 else 5.25, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [5, 300, 4096, 5000, 70000])
@pytest.mark.parametrize("kind", ["one id", "all empty", "two", "frequent", "descending", "first and last", "outside"])
def test_lookup_distributions(kind, n):
    """Runs that cross every kind of boundary: one id everywhere (all levels), runs cut by chunks, ids at both ends of the table, slots without an id."""
    n_codes, dim = 517, 20
    g = torch.Generator().manual_seed(n)
    i = torch.arange(n)
    ids = {"one id": torch.full((n,), 300), "all empty": torch.full((n,), -1), "two": i % 2 * 516, "frequent": torch.where(torch.rand(n, generator=g) < 0.9, 7, i % n_codes),
           "descending": (n - 1 - i) * n_codes // n, "first and last": torch.where(i < n // 3, 0, torch.where(i < n // 2, -1, 516)),
           "outside": torch.randint(-100, 700, (n,), generator=g)}[kind]
    table = torch.randn(n_codes, dim, generator=g).to(dev())
    check(ids.to(dev()), table, 0.5, None)
    check(ids.to(torch.int32).to(dev()), table, 1.0, torch.bfloat16)


@pytest.mark.gpu
def test_lookup_long_list_of_one_id_and_large_numbers():
    """1.3 million positions in four levels; a table whose offsets pass 2^32 bytes and whose ids need three radix passes."""
    table = torch.randn(3, 8, device=dev())
    ids = torch.full((1300000,), 1, device=dev())
    ids[5] = 2
    check(ids, table, 1.0, None)
    n_codes = (1 << 21) + 5
    big = torch.zeros(n_codes, 640, device=dev(), dtype=torch.bfloat16).requires_grad_(True)     # 2.7 GB: 1.3e9 elements
    at = torch.tensor([n_codes - 1, 0, n_codes - 1, 1 << 20, 77] + [n_codes - 2] * 5000, device=dev())
    with torch.no_grad():
        big[n_codes - 1] = 3.0
        big[n_codes - 2] = 2.0
    out = codes.lookup(at, big)
    assert bool((out[0] == 3).all()) and bool((out[2] == 3).all()) and not out[1].any() and bool((out[5:] == 2).all())
    d = torch.ones_like(out)
    d[2] = 0.5
    g, = torch.autograd.grad(out, big, d)
    assert bool((g[n_codes - 1] == 1.5).all()) and bool((g[0] == 1).all()) and bool((g[77] == 1).all()) and bool((g[1 << 20] == 1).all())
    assert bool((g[n_codes - 2] == 4992).all())                        # 5000 in bf16 (steps of 32)
    assert int(torch.count_nonzero(g.sum(1))) == 5


@pytest.mark.gpu
def test_lookup_shapes_strides_and_empty_batches():
    table = torch.randn(40, 12, device=dev())
    ids = torch.randint(0, 40, (6, 10), device=dev())
    assert torch.equal(codes.lookup(ids.t(), table), table[ids.t()])
    assert torch.equal(codes.lookup(ids[:, ::3], table[:, 3:9]), table[:, 3:9][ids[:, ::3]])       # rows 12 apart: copied first
    assert torch.equal(codes.lookup(torch.tensor(7, device=dev()), table), table[7])
    t = table.clone().requires_grad_(True)
    out = codes.lookup(ids[:0], t)
    assert out.shape == (0, 10, 12)
    g, = torch.autograd.grad(out, t, torch.zeros_like(out))
    assert g.shape == t.shape and not g.any()
    # a column slice of a gradient and an expanded one reach the kernel as they are
    out = codes.lookup(ids, t)
    g, = torch.autograd.grad(out.sum(), t)
    want, s, c = plain_grad(ids, torch.ones(6, 10, 12), 40, 1.0)
    assert torch.equal(g.cpu().double(), want)


@pytest.mark.gpu
def test_lookup_non_finite_values_stay_in_their_rows():
    table = torch.randn(9, 6, device=dev())
    table[4, 2] = float("inf")
    ids = torch.tensor([4, 1, 4, 3, -1], device=dev())
    t = table.clone().requires_grad_(True)
    out = codes.lookup(ids, t)
    assert bool(out[0, 2].isinf()) and int((~out.isfinite()).sum()) == 2
    d = torch.ones_like(out)
    d[4] = float("nan")                                                # the gradient of an empty slot reaches nothing
    d[1, 0] = float("inf")
    g, = torch.autograd.grad(out, t, d)
    assert bool(g[1, 0].isinf()) and int((~g.isfinite()).sum()) == 1


@pytest.mark.gpu
def test_lookup_verifies_ids_on_request(monkeypatch):
    monkeypatch.setattr(codes, "CHECK_IDS", True)
    table = torch.randn(4, 4, device=dev())
    codes.lookup(torch.tensor([3, -1], device=dev()), table)
    with pytest.raises(IndexError, match="id 4 in a table of 4"):
        codes.lookup(torch.tensor([1, 4], device=dev()), table)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [33, 3000, 9000])
def test_lookup_gradient_captured_and_replayed(n):
    """The plain calls inside a captured graph, replayed with other ids and other work between the replays."""
    table = torch.randn(700, 48, device=dev())
    ids, dout = torch.randint(0, 700, (n,), device=dev()), torch.randn(n, 48, device=dev())

    def step():
        t = table.detach().requires_grad_(True)
        out = codes.lookup(ids, t, 2.0)
        return out.detach(), torch.autograd.grad(out, t, dout)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for k in range(4):
        ids.copy_(torch.randint(-2, 700, (n,), device=dev()) // (1 + 300 * (k == 2)))
        dout.copy_(torch.randn(n, 48, device=dev()))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_lookup_two_streams_at_once():
    tables = [torch.randn(90, 64, device=dev()) for _ in range(2)]
    ids = [torch.randint(0, 90, (9000,), device=dev()) for _ in range(2)]
    dout = [torch.randn(9000, 64, device=dev()) for _ in range(2)]

    def step(i):
        t = tables[i].detach().requires_grad_(True)
        return torch.autograd.grad(codes.lookup(ids[i], t), t, dout[i])[0]
    want = [step(i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got.append((i, step(i)))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i, g in got)


@pytest.mark.gpu
def test_code_table_trains_with_the_one_launch_optimizer():
    from nvp_amd.optim import AdamW
    m = codes.CodeTable(30, 16, scale=4.0).to(dev())
    opt = AdamW(m.parameters(), lr=1e-2)
    ids = torch.arange(20, device=dev()).repeat(3)
    before = m.codes.detach().clone()
    m(ids).square().sum().backward()
    opt.step()
    moved = (m.codes.detach() - before).abs().amax(1)
    assert bool((moved[:20] > 0).all()) and bool((moved[20:] <= 1e-2 * 1e-2 * 1e-4 * 1.01).all())   # rows no id points to only decay


@pytest.mark.gpu
def test_lookup_is_differentiable_once_and_guards_what_it_saved():
    table = torch.randn(9, 5, device=dev(), requires_grad=True)
    ids = torch.tensor([1, 1, 8, -1], device=dev())
    out = codes.lookup(ids, table)
    dout = torch.ones_like(out, requires_grad=True)
    g, = torch.autograd.grad(out, table, dout, create_graph=True)
    assert torch.equal(g.detach()[1], torch.full((5,), 2.0, device=dev()))
    with pytest.raises(RuntimeError, match="once"):
        g.sum().backward()
    out = codes.lookup(ids, table)
    first, = torch.autograd.grad(out.sum(), table, retain_graph=True)
    second, = torch.autograd.grad(out.sum(), table)
    assert torch.equal(first, second)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(out.sum(), table)
    out = codes.lookup(ids, table)
    ids.fill_(0)                                                    # the ids belong to the recorded call
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(out.sum(), table)
    with torch.inference_mode():
        assert not codes.lookup(ids, table).requires_grad
    with pytest.raises(RuntimeError, match="HIP device"):
        codes.lookup(ids.cpu(), table)


@pytest.mark.gpu
@pytest.mark.parametrize("n,n_codes", [(4097, 3), (10000, 1), (20000, 1 << 20), (300000, 600)])
def test_lookup_gradient_bits_of_the_sort(n, n_codes):
    """Integers: sums are exact whatever their order, so every row has to come out right to the bit - one digit, two and three of them."""
    g = torch.Generator().manual_seed(n)
    ids = torch.randint(-1, n_codes, (n,), generator=g).to(dev())
    dout = torch.randint(-8, 9, (n, 8), generator=g).float().to(dev())
    t = torch.zeros(n_codes, 8, device=dev(), requires_grad=True)
    got, = torch.autograd.grad(codes.lookup(ids, t), t, dout)
    want, _, _ = plain_grad(ids, dout, n_codes, 1.0)
    assert torch.equal(got.cpu().double(), want)


@pytest.mark.gpu
def test_lookup_offsets_past_32_bits():
    """2.2e9 values out and back: integers below 2^24 in 32-bit sums, so the gradient is exact before its one rounding."""
    n, n_codes, dim = 2_200_000, 300, 1000
    ids = torch.randint(0, n_codes, (n,), device=dev())
    table = torch.randn(n_codes, dim, device=dev(), dtype=B16, requires_grad=True)
    out = codes.lookup(ids, table)
    assert all(torch.equal(out[a:a + 1000], table.detach()[ids[a:a + 1000]]) for a in (0, 2_147_400, n - 1000))
    dout = torch.randn(n, dim, device=dev(), dtype=B16).round_()
    got, = torch.autograd.grad(out, table, dout)
    want = torch.zeros(n_codes, dim, device=dev(), dtype=torch.float64)
    for a in range(0, n, 200_000):
        want.index_add_(0, ids[a:a + 200_000], dout[a:a + 200_000].double())
    assert torch.equal(got, want.to(B16))


@pytest.mark.gpu
def test_lookup_in_a_table_past_32_bits():
    n_codes, dim = 70_000, 40_001                                   # 2.8e9 values, rows that are not 16-byte aligned
    table = torch.randn(n_codes, dim, device=dev(), dtype=B16, requires_grad=True)
    ids = torch.tensor([n_codes - 1, 0, 53_700, n_codes - 1, -1], device=dev())
    out = codes.lookup(ids, table)
    assert torch.equal(out[:4], table.detach()[ids[:4]]) and not out[4].any()
    dout = torch.randint(-8, 9, (5, dim), device=dev()).to(B16)
    got, = torch.autograd.grad(out, table, dout)
    assert torch.equal(got[n_codes - 1], dout[0] + dout[3]) and torch.equal(got[0], dout[1]) and torch.equal(got[53_700], dout[2])
    rows = torch.cat([got[a:a + 10_000].ne(0).any(1) for a in range(0, n_codes, 10_000)]).nonzero().flatten()
    assert rows.tolist() == [0, 53_700, n_codes - 1]


@pytest.mark.gpu
@pytest.mark.parametrize("table_dtype,dtype", PAIRS)
@pytest.mark.parametrize("n,n_codes,dim", [(131072, 1, 32), (140001, 600, 32), (139999, 1023, 7), (135171, 1024, 33), (150000, 2, 256), (131073, 37, 257), (133333, 300, 3),
                                           (262145, 900, 8), (139265, 64, 255), (200000, 5, 1)])
def test_lookup_many_rows_of_few_codes(n, n_codes, dim, table_dtype, dtype):
    g = torch.Generator().manual_seed(n + dim)
    ids = torch.randint(0, n_codes, (n,), generator=g)
    ids[torch.rand(n, generator=g) < 0.05] = -1
    check(ids.to(dev()), torch.randn(n_codes, dim, generator=g).to(table_dtype).to(dev()), 1.5, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["one", "none", "sorted", "most", "chunks", "pairs"])
def test_lookup_few_codes_distributions(kind):
    """Integers, so that every order of the sums is exact: one id everywhere, none, whole chunks of one id, runs over every edge between teams."""
    n, n_codes, dim = 300_001, 600, 20
    g = torch.Generator().manual_seed(1)
    ids = {"one": torch.full((n,), 599), "none": torch.full((n,), -1), "sorted": torch.arange(n) * n_codes // n,
           "most": torch.where(torch.rand(n, generator=g) < 0.99, 3, torch.randint(0, n_codes, (n,), generator=g)),
           "chunks": torch.arange(n) // 4096 * 7 % n_codes, "pairs": torch.arange(n) // 2 % n_codes}[kind].to(dev())
    dout = torch.randint(-8, 9, (n, dim), generator=g).float().to(dev())
    t = torch.zeros(n_codes, dim, device=dev(), requires_grad=True)
    got, = torch.autograd.grad(codes.lookup(ids, t), t, dout)
    assert torch.equal(got.cpu().double(), plain_grad(ids, dout, n_codes, 1.0)[0])


@pytest.mark.gpu
def test_lookup_few_codes_captured_and_on_two_streams():
    n, table = 270_000, torch.randn(500, 24, device=dev())
    ids, dout = torch.randint(0, 500, (n,), device=dev()), torch.randn(n, 24, device=dev())

    def step():
        t = table.detach().requires_grad_(True)
        return torch.autograd.grad(codes.lookup(ids, t, 2.0), t, dout)[0]
    want = step()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for st in streams:
            with torch.cuda.stream(st):
                got.append(step())
    torch.cuda.synchronize()
    assert all(torch.equal(a, want) for a in got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        ids.copy_(torch.randint(-2, 500, (n,), device=dev()) // (1 + 300 * (k == 2)))
        dout.copy_(torch.randn(n, 24, device=dev()))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [5, 700, 1024, 1025, 5000, 70000, 600000])
@pytest.mark.parametrize("kind", ["one id", "all empty", "two", "frequent", "descending", "first and last", "outside"])
def test_lookup_distributions_of_many_codes(kind, n):
    """The same over the whole batch's sort: integers, so that sums are exact in any order."""
    n_codes, dim = 1517, 20
    g = torch.Generator().manual_seed(n)
    i = torch.arange(n)
    ids = {"one id": torch.full((n,), 300), "all empty": torch.full((n,), -1), "two": i % 2 * 1516, "frequent": torch.where(torch.rand(n, generator=g) < 0.9, 7, i % n_codes),
           "descending": (n - 1 - i) * n_codes // n, "first and last": torch.where(i < n // 3, 0, torch.where(i < n // 2, -1, 1516)),
           "outside": torch.randint(-100, 1700, (n,), generator=g)}[kind]
    for dt in (torch.int64, torch.int32):
        dout = torch.randint(-8, 9, (n, dim), generator=g).float().to(dev())
        t = torch.zeros(n_codes, dim, device=dev(), requires_grad=True)
        got, = torch.autograd.grad(codes.lookup(ids.to(dt).to(dev()), t), t, dout)
        assert torch.equal(got.cpu().double(), plain_grad(ids, dout, n_codes, 1.0)[0])


@pytest.mark.gpu
@pytest.mark.parametrize("table_dtype,dtype", PAIRS)
@pytest.mark.parametrize("n,n_codes,dim", [(900, 5, 129), (1300000, 3, 136), (262145, 100, 65), (262144, 1023, 128), (1000, 1024, 20), (1500, 1, 200), (4096, 3000, 513)])
def test_lookup_at_the_borders_of_the_two_ways(n, n_codes, dim, table_dtype, dtype):
    g = torch.Generator().manual_seed(n + dim)
    check(torch.randint(-1, n_codes, (n,), generator=g).to(dev()), torch.randn(n_codes, dim, generator=g).to(table_dtype).to(dev()), 1.5, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("table_dtype,dtype", PAIRS)
@pytest.mark.parametrize("n,n_codes,dim", [(1, 1025, 1), (9, 40, 301), (513, 5000, 333), (1024, 4096, 129), (1025, 4100, 130), (1025, 4099, 130), (3000, 200000, 17), (2049, 1 << 21, 5)])
def test_lookup_mostly_empty_tables(n, n_codes, dim, table_dtype, dtype):
    """Zeros written beside the sort (and behind it, just short of that): odd sizes, so that the last bytes are fewer than one access."""
    g = torch.Generator().manual_seed(n + dim)
    junk = torch.full((n_codes, dim), float("nan"), device=dev(), dtype=table_dtype)       # the allocator hands this memory out again: what is not written shows
    del junk
    check(torch.randint(-1, n_codes, (n,), generator=g).to(dev()), torch.randn(n_codes, dim, generator=g).to(table_dtype).to(dev()), 1.5, dtype)


def test_a_missing_binding_is_an_error(monkeypatch, tmp_path):
    monkeypatch.setattr(L, "_binding", None)
    monkeypatch.setattr(L, "_HERE", str(tmp_path))
    with pytest.raises(RuntimeError, match="the binding is not built"):
        codes.lookup(torch.zeros(3, dtype=torch.int64), torch.zeros(4, 5))


def test_lookup_refuses_forward_mode_tangents():
    from torch.autograd import forward_ad
    with forward_ad.dual_level():
        table = forward_ad.make_dual(torch.zeros(4, 5), torch.ones(4, 5))
        with pytest.raises(NotImplementedError, match="lookup has no forward-mode derivative"):
            codes.lookup(torch.zeros(3, dtype=torch.int64), table)
        with pytest.raises(RuntimeError, match="HIP device"):            # without its tangent: taken, and what is refused is the device
            codes.lookup(torch.zeros(3, dtype=torch.int64), forward_ad.unpack_dual(table).primal)


@pytest.mark.gpu
def test_lookup_refuses_a_gradient_with_a_tangent():
    from torch.autograd import forward_ad
    table = torch.randn(4, 5, device=dev(), requires_grad=True)
    out = codes.lookup(torch.tensor([1, 1, 3], device=dev()), table)
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="the gradient of lookup has no forward-mode derivative"):
            torch.autograd.grad(out, table, forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out)))
        with pytest.raises(NotImplementedError):
            codes.lookup(torch.tensor([1], device=dev()), forward_ad.make_dual(table, torch.ones_like(table)))


@pytest.mark.gpu
def test_lookup_of_more_rows_than_one_launch_takes():
    """16 rows a workgroup of 256 threads: 2^28 rows are 2^32 threads."""
    n, dim = (1 << 28) + 1000, 257
    if torch.cuda.mem_get_info()[0] < 160 << 30:
        pytest.skip("needs 140 GiB of device memory")
    table = torch.randn(50, dim, device=dev(), dtype=B16)
    ids = torch.randint(-1, 50, (n,), device=dev(), dtype=torch.int32)
    out = codes.lookup(ids, table)
    for a in (0, (1 << 28) - 600, (1 << 28) - 16, n - 1000):
        i = ids[a:a + 1000].long()
        assert torch.equal(out[a:a + 1000], table[i.clamp(min=0)] * (i >= 0)[:, None]), a
    del out, ids
    torch.cuda.empty_cache()


# ---- the whole batch's sort (1024 codes or more, or wide rows), where fewer codes go chunk by chunk ------------------------------------------------
# one workgroup's sort (n <= 1024) and radix passes, one or two levels of sums; from codes >= 4 n on the zeros are written beside the sort
SORTED = [(700, 1500, 48), (9000, 1500, 48), (70000, 5000, 32), (700, 4000, 48), (9000, 40000, 130), (70000, 300000, 16)]


def sorted_step(ids, table, dout):
    t = table.detach().requires_grad_(True)
    out = codes.lookup(ids, t, 2.0)
    return out.detach(), torch.autograd.grad(out, t, dout)[0]


@pytest.mark.gpu
@pytest.mark.parametrize("n,n_codes,dim", SORTED)
def test_lookup_gradient_by_the_whole_sort_captured_and_replayed(n, n_codes, dim):
    table = torch.randn(n_codes, dim, device=dev())
    ids, dout = torch.randint(0, n_codes, (n,), device=dev()), torch.randn(n, dim, device=dev())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        sorted_step(ids, table, dout)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = sorted_step(ids, table, dout)
    for k in range(4):
        ids.copy_(torch.randint(-2, n_codes, (n,), device=dev()) // (1 + 1000 * (k == 2)))
        dout.copy_(torch.randn(n, dim, device=dev()))
        got[1].fill_(float("nan"))                                  # rows that a replay leaves out would show
        graph.replay()
        want = sorted_step(ids, table, dout)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        grad, s, c = plain_grad(ids, dout, n_codes, 2.0)
        assert bool(((got[1].double().cpu() - grad).abs() <= (c + 1) * 2.0 ** -24 * s * (1 + E) + E * grad.abs()).all())


@pytest.mark.gpu
@pytest.mark.parametrize("n,n_codes,dim", SORTED)
def test_lookup_gradient_by_the_whole_sort_on_two_streams(n, n_codes, dim):
    tables = [torch.randn(n_codes, dim, device=dev()) for _ in range(2)]
    ids = [torch.randint(0, n_codes, (n,), device=dev()) for _ in range(2)]
    dout = [torch.randn(n, dim, device=dev()) for _ in range(2)]
    want = [sorted_step(ids[i], tables[i], dout[i])[1] for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got.append((i, sorted_step(ids[i], tables[i], dout[i])[1]))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i, g in got)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["one id", "random", "two", "sorted"])
@pytest.mark.parametrize("n,n_codes,dim", [(800_000, 5000, 32), (1_000_000, 70_000, 24), (1_300_000, 2000, 8), (300_000, 1100, 260)])
def test_lookup_gradient_of_a_long_list_by_the_whole_sort(n, n_codes, dim, kind):
    """The first two have three levels of sums, the third into the first one's list: with 32 entries a team, 800 000 positions leave a list of 50 000 partial rows, that one
    of 3126, more than the last launch takes, that one of 196.  Integers: exact in any order."""
    g = torch.Generator().manual_seed(n)
    i = torch.arange(n)
    ids = {"one id": torch.full((n,), n_codes - 1), "random": torch.randint(-1, n_codes, (n,), generator=g), "two": i % 2 * (n_codes - 1), "sorted": i * n_codes // n}[kind].to(dev())
    dout = torch.randint(-8, 9, (n, dim), generator=g).float().to(dev())
    t = torch.zeros(n_codes, dim, device=dev(), requires_grad=True)
    got, = torch.autograd.grad(codes.lookup(ids, t), t, dout)
    assert torch.equal(got.double().cpu(), plain_grad(ids, dout, n_codes, 1.0)[0])
