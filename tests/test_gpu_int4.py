"""GPU tests of the 4-bit linear against the formula in 64 bits.

Tolerances: an FP32 sum of K products is off by at most (K + 32) 2^-24 of the
sum of their magnitudes, where the magnitudes are those that the kernels add:
|x| (|scale| q' + |offset|) with q' up to 143, because up to 16 rows multiply by
128 + q (32 rows over at most 8,192 columns); over more rows the weights are rounded to bf16, half a step (2^-8) of
each.  The result is rounded once more."""

from __future__ import annotations

import pytest

from conftest import pkg, submodule

pytestmark = pytest.mark.gpu

STEP, HALF = 2.0**-24, 2.0**-8
FEW = 16  # rows up to which the codes themselves are multiplied; 32 over at most 8,192 columns


def _problem(rows, n, k, group, offsets=True, f32=False, bias=False, seed=0, lead=None):
    import torch

    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    t = torch.float32 if f32 else torch.bfloat16
    codes = torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = ((torch.rand(n, k // group, generator=g, device="cuda") + 0.5) * 0.01).to(t)
    off = (torch.randn(n, k // group, generator=g, device="cuda") * 0.05 - 0.07).to(t) if offsets else None
    b = torch.randn(n, generator=g, device="cuda").to(t) if bias else None
    x = (torch.randn(*(lead or (rows,)), k, generator=g, device="cuda") + 0.1).to(torch.bfloat16)
    return x, codes, scales, off, b


def _check(problem, y=None):
    import torch

    x, codes, scales, off, bias = problem
    n, k = codes.shape[0], 2 * codes.shape[1]
    y = pkg().int4_linear(*problem) if y is None else y
    assert y.dtype == torch.bfloat16 and y.shape == (*x.shape[:-1], n)
    group = k // scales.shape[1]
    q = torch.stack([codes & 15, codes >> 4], 2).view(n, k).double()
    s = scales.double().repeat_interleave(group, 1)
    o = -8 * s if off is None else off.double().repeat_interleave(group, 1)
    w = s * q + o
    v = x.double().reshape(-1, k)
    b = 0 if bias is None else bias.double()
    want = v @ w.t() + b
    mag = v.abs() @ (s * 143 + o.abs() + 128 * s).t()
    err = (k + 32) * STEP * mag
    if v.shape[0] > (32 if n <= 8192 else FEW):
        err = err + HALF * (v.abs() @ w.abs().t())
    got = y.double().view(want.shape)
    bad = ~((got - want).abs() <= HALF * (want.abs() + err) + err)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4], got[bad][:4], want[bad][:4])
    if want.numel() >= 4096:  # two roundings, each rms 2^-8 / sqrt(3) or less; twice their sum
        rms = (want - b).square().mean().sqrt() + (0 if bias is None else b.square().mean().sqrt())
        assert (got - want).square().mean().sqrt() <= 2 * HALF * rms
    return y


@pytest.mark.parametrize("rows", [1, 2, 3, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 300])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_rows_and_groups(dev, rows, group):
    _check(_problem(rows, 200, 512, group, seed=rows))


@pytest.mark.parametrize("n", [1, 2, 3, 5, 15, 16, 17, 63, 66, 127, 129, 255, 256, 257, 1000, 4096])
@pytest.mark.parametrize("rows", [1, 5, 16, 40, 200])
def test_output_widths(dev, n, rows):
    _check(_problem(rows, n, 256, 64, bias=True, seed=n))


@pytest.mark.parametrize("k, group", [(32, 32), (64, 32), (96, 32), (64, 64), (160, 32), (192, 64), (128, 128), (384, 128),
                                      (416, 32), (1088, 64), (4096, 64), (7168, 128), (8192, 32), (11008, 128),
                                      (18432, 64)])
@pytest.mark.parametrize("rows", [1, 4, 16, 17, 130])
def test_contractions(dev, k, group, rows):
    _check(_problem(rows, 72, k, group, seed=k))


@pytest.mark.parametrize("offsets", [False, True])
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("rows", [1, 13, 100])
def test_tables(dev, offsets, f32, bias, rows):
    _check(_problem(rows, 136, 640, 32, offsets, f32, bias))


@pytest.mark.parametrize("rows, n, k, group", [(1, 4096, 4096, 64), (16, 4096, 7168, 128), (300, 1536, 4096, 32),
                                               (2048, 4096, 1024, 128), (1, 30000, 512, 64), (5000, 96, 128, 32)])
def test_larger(dev, rows, n, k, group):
    _check(_problem(rows, n, k, group))


# 256, 512 and 1,024 workgroups, x of 32 and 48 KB and past it, tables of every kind
@pytest.mark.parametrize("n", [4097, 8190, 8193, 16383, 16385])
@pytest.mark.parametrize("rows, k, group", [(1, 1056, 32), (9, 2560, 128), (16, 1600, 64), (16, 2048, 32), (2, 8320, 64),
                                           (17, 1056, 32), (24, 8320, 128), (32, 1600, 64)])
@pytest.mark.parametrize("f32", [False, True])
def test_many_workgroups(dev, n, rows, k, group, f32):
    _check(_problem(rows, n, k, group, offsets=n % 2 == 1, f32=f32))


def test_every_code_in_every_place(dev):
    """One-hot rows read each weight of a matrix that holds each code in each
    column: q, scale and offset chosen exact in bf16."""
    import torch

    k, n = 128, 16
    q = (torch.arange(n, device=dev)[:, None] + torch.arange(k, device=dev)) % 16
    codes = (q[:, 0::2] | (q[:, 1::2] << 4)).to(torch.uint8)
    scales = torch.tensor([1.0, 0.5, 2.0, 0.25], device=dev).repeat(n, 1).to(torch.bfloat16)
    off = torch.tensor([-4.0, 1.0, -16.0, 0.0], device=dev).repeat(n, 1).to(torch.bfloat16)
    want = (q * scales.float().repeat_interleave(32, 1) + off.float().repeat_interleave(32, 1)).t()
    x = torch.eye(k, device=dev, dtype=torch.bfloat16)
    assert torch.equal(pkg().int4_linear(x, codes, scales, off).float(), want)
    for first in range(0, k, 16):
        assert torch.equal(pkg().int4_linear(x[first:first + 16], codes, scales, off).float(), want[first:first + 16])
    for one in (0, 1, 31, 32, 77, 127):
        assert torch.equal(pkg().int4_linear(x[one], codes, scales, off).float(), want[one])


def test_nan_and_infinity_stay_in_their_rows(dev):
    import torch

    for rows in (4, 20, 40):
        p = _problem(rows, 80, 256, 64)
        clean = pkg().int4_linear(*p)
        x = p[0].clone()
        x[1, 3], x[2, 100], x[3] = float("nan"), float("inf"), 2.0**120  # row 3: 143 times its sum is infinite
        y = pkg().int4_linear(x, *p[1:])
        q = (p[1][:, 50] & 15).float()
        w = q * p[2][:, 1].float() + p[3][:, 1].float()  # column 100's weights: what the infinity meets
        assert y[1].isnan().all() and torch.equal(y[2].float(), float("inf") * w)
        _check((x[3:4].expand(rows, 256).contiguous(), *p[1:]))
        keep = [r for r in range(rows) if r not in (1, 2, 3)]
        assert torch.equal(y[keep], clean[keep])


def test_shapes_views_and_empty(dev):
    import torch

    M = pkg()
    x, codes, scales, off, bias = _problem(12, 40, 128, 64, bias=True)
    want = M.int4_linear(x, codes, scales, off, bias)
    assert torch.equal(M.int4_linear(x.view(3, 4, 128), codes, scales, off, bias), want.view(3, 4, 40))
    flat = torch.empty(12 * 128 + 1, device=dev, dtype=torch.bfloat16)
    flat[1:].view(12, 128).copy_(x)
    store = torch.empty(40 * 64 + 3, device=dev, dtype=torch.uint8)
    store[3:].view(40, 64).copy_(codes)
    assert torch.equal(M.int4_linear(flat[1:].view(12, 128), store[3:].view(40, 64), scales, off, bias), want)
    assert torch.equal(M.int4_linear(x.t().contiguous().t(), codes.t().contiguous().t(), scales.t().contiguous().t(),
                                     off.t().contiguous().t(), bias), want)
    assert torch.equal(M.int4_linear(x[3], codes, scales, off, bias), M.int4_linear(x[3:4], codes, scales, off, bias)[0])
    assert M.int4_linear(x[:0], codes, scales, off, bias).shape == (0, 40)
    wide = torch.cat([codes, codes])
    assert torch.equal(M.int4_linear(x, wide[:40], scales, off, bias), want)


def test_runs_repeat_and_bias_adds_nothing_else(dev):
    import torch

    for rows in (1, 16, 70, 500):
        p = _problem(rows, 264, 2048, 64)
        y = pkg().int4_linear(*p)
        for _ in range(3):
            assert torch.equal(pkg().int4_linear(*p), y)
        zero = torch.zeros(264, device=dev, dtype=torch.bfloat16)
        assert torch.equal(pkg().int4_linear(*p[:4], zero), y)


@pytest.mark.parametrize("rows", [1, 16, 60, 300])
def test_other_stream_and_captured_graph(dev, rows):
    import torch

    M = pkg()
    p = list(_problem(rows, 200, 1024, 64, bias=True))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        M.int4_linear(*p)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            got = M.int4_linear(*p)
    torch.cuda.current_stream().wait_stream(s)
    for k in range(3):
        for t, v in zip(p, _problem(rows, 200, 1024, 64, bias=True, seed=9 + k)):
            t.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, M.int4_linear(*p)), k


def test_modules(dev):
    """Int4Linear from a linear, and the 4-bit MLP of a GatedMLP, against the
    weights they hold, in the MLP with the package's own bf16 SwiGLU."""
    import torch

    M = pkg()
    fp8 = submodule("fp8")
    lin = torch.nn.Linear(256, 120, device=dev).to(torch.bfloat16)
    for symmetric in (False, True):
        layer = M.Int4Linear.from_linear(lin, group_size=32, symmetric=symmetric)
        x = torch.randn(9, 256, device=dev).to(torch.bfloat16)
        _check((x, layer.weight, layer.scales, layer.offsets, layer.bias), layer(x))
        again = M.Int4Linear(256, 120, group_size=32, symmetric=symmetric, bias=True, device=dev)
        again.load_state_dict(layer.state_dict())
        assert torch.equal(again(x), layer(x))
    mlp = M.GatedMLP(256, 128, limit=2.0, device=dev)
    small = mlp.to_int4(group_size=64)
    for rows in (1, 30):
        x = torch.randn(rows, 256, device=dev).to(torch.bfloat16)
        joined = small.gate_up_proj(x)
        h = fp8.swiglu(joined[:, :128], joined[:, 128:], 2.0)
        assert torch.equal(small(x), small.down_proj(h))
        compiled = torch.compile(small, backend="aot_eager", fullgraph=True)
        assert torch.equal(compiled(x), small(x))
    assert small(torch.randn(2, 3, 256, device=dev).to(torch.bfloat16)).shape == (2, 3, 256)


def test_refusals(dev):
    import torch

    M = pkg()
    x, c, s, o, b = _problem(4, 40, 128, 64, bias=True)
    bad = [
        lambda: M.int4_linear(x.float(), c, s), lambda: M.int4_linear(x, c.int(), s), lambda: M.int4_linear(x, c[0], s),
        lambda: M.int4_linear(x[:, :64], c, s), lambda: M.int4_linear(x, c, s.half()), lambda: M.int4_linear(x, c, s[:8]),
        lambda: M.int4_linear(x, c, s[:, :0]), lambda: M.int4_linear(x, c, s.repeat(1, 4)),
        lambda: M.int4_linear(x, c, s, o.float()), lambda: M.int4_linear(x, c, s, o[:8]), lambda: M.int4_linear(x, c, s, o, b[:8]),
        lambda: M.int4_linear(x, c, s, o, b.float()), lambda: M.int4_linear(x, c[:0], s[:0]), lambda: M.int4_linear(x, c, s.cpu()),
        lambda: M.int4_linear(x[0, 0], c, s),
    ]
    for k, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {k} was not refused")
    with pytest.raises(RuntimeError):  # no gradient is claimed where there is none
        M.int4_linear(x.requires_grad_(), c, s).sum().backward()


@pytest.mark.parametrize("rows", [1, 16, 40, 200])
def test_offsets_past_32_bits(dev, rows):
    """More than 2^32 codes: the last output columns are those of a call on
    their rows alone."""
    import torch

    M = pkg()
    n, k, tail = 70_000, 1 << 16, 24
    assert n * k > 2**32
    p = _problem(rows, tail, k, 128, bias=True)
    codes = torch.zeros(n, k // 2, device=dev, dtype=torch.uint8)
    scales = torch.ones(n, k // 128, device=dev, dtype=torch.bfloat16)
    off, bias = torch.zeros_like(scales), torch.zeros(n, device=dev, dtype=torch.bfloat16)
    for big, small in ((codes, p[1]), (scales, p[2]), (off, p[3]), (bias, p[4])):
        big[-tail:] = small
    y = M.int4_linear(p[0], codes, scales, off, bias)
    assert (y[:, :-tail] == 0).all()
    _check(p, y[:, -tail:].contiguous())


def test_mlp_without_a_limit(dev):
    import torch

    M, fp8 = pkg(), submodule("fp8")
    small = M.GatedMLP(128, 64, device=dev).to_int4(group_size=32, symmetric=True)
    x = (8 * torch.randn(7, 128, device=dev)).to(torch.bfloat16)
    joined = small.gate_up_proj(x)
    assert torch.equal(small(x), small.down_proj(fp8.swiglu(joined[:, :64], joined[:, 64:], float("inf"))))
