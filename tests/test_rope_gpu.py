"""Rotary positions (b200moe_op_rope) against the formula in 64 bits.

Tolerance: the turn's angle is reduced in double to an error below 1e-9; its fp32 sine and cosine are within 2 ulp of 2^-24, the two products and their sum add three
roundings: |error| <= 2^-22 (|x0| + |x1|) before the output's rounding of half a step (2^-24, bf16 2^-8) of the value."""
import numpy as np
import pytest
import torch

from edge0_b200.capi import B200MoeError

pytestmark = pytest.mark.gpu


def formula(x, pos, n_rot, base, sections, interleaved, adjacent, inverse):
    """x [T, H, D], pos [axes, T] -> float64 (result, sum of the sizes of each pair's values)"""
    x = np.asarray(x, np.float64)
    half, A = n_rot // 2, len(sections)
    y, size = x.copy(), np.abs(x)
    bounds = np.cumsum(sections)
    for i in range(half):
        a = (i % A if i < A * sections[i % A] else 0) if interleaved else int(np.searchsorted(bounds, i, side="right"))
        w = np.asarray(pos[a], np.float64) * base ** (-2.0 * i / n_rot) * (-1.0 if inverse else 1.0)
        p, q = (2 * i, 2 * i + 1) if adjacent else (i, i + half)
        c, s = np.cos(w)[:, None], np.sin(w)[:, None]
        y[..., p], y[..., q] = x[..., p] * c - x[..., q] * s, x[..., p] * s + x[..., q] * c
        size[..., p] = size[..., q] = np.abs(x[..., p]) + np.abs(x[..., q])
    return y, size


def close(got, want, size):
    half_step = 2.0 ** (-8 if got.dtype == torch.bfloat16 else -24)
    err = np.abs(got.double().cpu().numpy() - want)
    assert (err <= half_step * np.abs(want) * 1.01 + 2.0 ** -22 * size + 1e-37).all(), float((err - half_step * np.abs(want)).max())


def inputs(T, H, D, dtype, axes, seed=0, far=1 << 20):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((T, H, D), generator=g).to(dtype)
    pos = torch.randint(-far, far, (axes, T), generator=g, dtype=torch.int32)
    return x, pos


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,H,D,n_rot,sections,interleaved,adjacent", [
    (1, 1, 128, 128, [64], False, False),
    (1, 36, 128, 128, [64], False, True),
    (3, 5, 64, 64, [32], False, False),
    (17, 3, 256, 256, [128], False, False),
    (300, 2, 128, 64, [32], False, False),          # half of a head turns
    (65, 2, 128, 64, [32], False, True),
    (33, 2, 80, 80, [40], False, False),            # not a power of two
    (9, 2, 66, 66, [33], False, False),             # no vectors: 33 pairs
    (9, 2, 66, 6, [3], False, True),
    (9, 2, 128, 2, [1], False, False),              # one pair
    (40, 3, 128, 128, [24, 20, 20], False, False),
    (40, 3, 128, 128, [24, 20, 20], True, False),
    (40, 3, 128, 128, [24, 20, 20], True, True),
    (21, 2, 64, 64, [8, 0, 20, 4], False, False),   # an axis without pairs
    (21, 2, 64, 32, [8, 8], True, False),
    (1201, 4, 128, 128, [16, 24, 24], False, False),
])
def test_against_the_formula(gpu_ctx, dtype, T, H, D, n_rot, sections, interleaved, adjacent):
    x, pos = inputs(T, H, D, dtype, len(sections), seed=T + D)
    for inverse in (False, True):
        y = gpu_ctx.rope(x.cuda(), pos.cuda(), base=1e6, n_rot=n_rot, sections=sections, interleaved=interleaved, adjacent=adjacent, inverse=inverse)
        close(y, *formula(x.double(), pos, n_rot, 1e6, sections, interleaved, adjacent, inverse))
        assert torch.equal(y[..., n_rot:].cpu(), x[..., n_rot:])


@pytest.mark.parametrize("base", [1e4, 5e5, 1.0, 0.5])
def test_far_positions_and_other_bases(gpu_ctx, base):
    x, _ = inputs(6, 2, 128, torch.float32, 1)
    pos = torch.tensor([0, 1, -1, 2 ** 31 - 1 if base >= 1 else 1000, 123456789 if base >= 1 else 77, -(2 ** 24) if base >= 1 else -5], dtype=torch.int32)
    y = gpu_ctx.rope(x.cuda(), pos.cuda(), base=base)
    want, size = formula(x.double(), pos[None], 128, base, [64], False, False, False)
    # 2^31 turns' worth of radians: numpy's own angle is good to 2^-53 * 2^31 there
    err = np.abs(y.double().cpu().numpy() - want)
    assert (err <= (2.0 ** -21 + 2e-6) * size).all()
    assert torch.equal(y[0].cpu(), x[0])                # position 0 turns nothing


def test_slices_strides_and_in_place(gpu_ctx):
    T, H, D = 19, 6, 128
    g = torch.Generator().manual_seed(4)
    qkv = torch.randn((T, H + 4, D), generator=g).to(torch.bfloat16)
    pos = torch.randint(0, 5000, (T,), generator=g, dtype=torch.int32)
    want, size = formula(qkv[:, :H].double(), pos[None], D, 1e6, [64], False, False, False)
    dev = qkv.cuda()
    before = dev.clone()
    y = gpu_ctx.rope(dev[:, :H], pos.cuda())
    close(y, want, size)
    assert torch.equal(dev, before)
    z = gpu_ctx.rope(dev[:, :H], pos.cuda(), out=dev[:, :H])
    assert z.data_ptr() == dev.data_ptr()
    assert torch.equal(dev[:, :H], y) and torch.equal(dev[:, H:], before[:, H:])
    # in place with values behind the turned ones
    half = before.clone()
    gpu_ctx.rope(half[:, :H], pos.cuda(), n_rot=64, out=half[:, :H])
    assert torch.equal(half[..., 64:], before[..., 64:])
    close(half[:, :H], *formula(qkv[:, :H].double(), pos[None], 64, 1e6, [32], False, False, False))
    # heads before tokens, and rows that start anywhere (pair by pair)
    t = before[:, :H].transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(gpu_ctx.rope(t, pos.cuda()), y)
    odd = torch.zeros(T * H * D + 1, dtype=torch.bfloat16, device="cuda")[1:].view(T, H, D)
    odd.copy_(before[:, :H])
    assert torch.equal(gpu_ctx.rope(odd, pos.cuda(), out=torch.empty(T * H * D + 1, dtype=torch.bfloat16, device="cuda")[1:].view(T, H, D)), y)


def test_inverse_is_the_gradient(gpu_ctx):
    """d(sum g . rope(x)) / dx = rope^-1(g), by the formula's transpose and by differences."""
    x, pos = inputs(5, 2, 64, torch.float32, 2, far=300)
    g = torch.randn((5, 2, 64), generator=torch.Generator().manual_seed(8))
    kw = dict(base=1e4, sections=[20, 12], interleaved=False)
    back = gpu_ctx.rope(g.cuda(), pos.cuda(), inverse=True, **kw).double().cpu()
    step = torch.randn(x.shape, generator=torch.Generator().manual_seed(9))
    f = lambda t: float((gpu_ctx.rope(t.cuda(), pos.cuda(), **kw).double().cpu() * g.double()).sum())
    # rope is linear: a difference over a whole step is the derivative; 640 values of size 1 with errors of 2^-22 each
    assert abs((f(x + step) - f(x)) - float((back * ((x + step).double() - x.double())).sum())) < 640 * 4 * 2.0 ** -20
    there = gpu_ctx.rope(gpu_ctx.rope(x.cuda(), pos.cuda(), **kw), pos.cuda(), inverse=True, **kw).cpu()
    assert (there - x).abs().max() < 2.0 ** -19 * 5


def test_graph_stream_and_empty(gpu_ctx):
    x, pos = inputs(7, 3, 128, torch.bfloat16, 1)
    x, pos = x.cuda(), pos[0].cuda()
    want = gpu_ctx.rope(x, pos)
    s = torch.cuda.Stream()
    out = torch.empty_like(x)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        gpu_ctx.rope(x, pos, out=out)
    s.synchronize()
    assert torch.equal(out, want)
    graph = torch.cuda.CUDAGraph()
    out.zero_()
    with torch.cuda.graph(graph):
        gpu_ctx.rope(x, pos, out=out)
    pos += 11
    graph.replay()
    assert torch.equal(out, gpu_ctx.rope(x, pos))
    assert gpu_ctx.rope(x[:0], pos[:0]).shape == (0, 3, 128)
    nan = x.clone()
    nan[0, 0, 0], nan[1, 1, 5] = float("nan"), float("inf")
    y = gpu_ctx.rope(nan, pos)
    bad = torch.zeros_like(x, dtype=torch.bool)
    bad[0, 0, [0, 64]], bad[1, 1, [5, 69]] = True, True
    assert torch.equal(~torch.isfinite(y), bad)
    with pytest.raises(B200MoeError):
        gpu_ctx.rope(x, pos, sections=[63])
    with pytest.raises(ValueError):
        gpu_ctx.rope(x, pos.long())
    with pytest.raises(ValueError):
        gpu_ctx.rope(x, pos[:3])
    with pytest.raises(ValueError):
        gpu_ctx.rope(x.cpu(), pos)
    with pytest.raises(ValueError):
        gpu_ctx.rope(x, pos.cpu())
    with pytest.raises(TypeError):
        gpu_ctx.rope(x.half(), pos)
