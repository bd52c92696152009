"""The cache that is quantised as it is written (b200moe_kv_write, b200moe_kv_read): every held value against the definition in 64 bits,
bit for bit, and what lies around the written rows."""
import numpy as np
import pytest
import torch

from edge0_b200.capi import B200MoeError
from edge0_b200.kv_cache import KvCache

pytestmark = pytest.mark.gpu


def held(x, kind):
    """float32 values that a cache stands for: x float32 numpy [..., D]"""
    if kind == "bf16":
        return torch.from_numpy(x).to(torch.bfloat16).float().numpy()
    n, top = (x.shape[-1], 127) if kind == "q8" else (32, 7)
    g = x.reshape(x.shape[:-1] + (-1, n))
    with np.errstate(all="ignore"):
        d = np.abs(g).max(-1, keepdims=True).astype(np.float32) / np.float32(top)     # one IEEE division
        if kind == "q4":
            d = torch.from_numpy(d).to(torch.bfloat16).float().numpy()
        code = np.where(d > 0, np.rint(g.astype(np.float64) / np.where(d > 0, d, 1).astype(np.float64)), 0)
        y = np.clip(code, -top, top).astype(np.float32) * d
        y = np.where(np.isfinite(g).all(-1, keepdims=True), y, np.float32("nan"))
    return y.reshape(x.shape).astype(np.float32)


def same(a, b):
    return bool(((a == b) | (torch.isnan(a) & torch.isnan(b))).all())


def make(gpu_ctx, kind, D, page=16, n_pages=9, heads=3):
    return KvCache(gpu_ctx, kind=kind, n_pages=n_pages, page_size=page, n_head_kv=heads, head_dim=D)


def hard_rows(T, H, D, dtype, seed):
    """Rows with values on the borders between codes, of every size, zeros, and rows that hold what cannot be quantised."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((T, H, D)).astype(np.float32)
    x[0] = 0
    if T > 1:
        x[1] = rng.integers(-14, 15, (H, D)) / 2.0                     # halves of whole steps for d = 1
        x[1, :, ::32] = 7
    if T > 2:
        x[2] = rng.integers(-254, 255, (H, D)) / 2.0
        x[2, :, 0] = 127
    if T > 3:
        x[3] *= np.float32(1e-38)
        x[3, 0] *= np.float32(1e-4)                                     # subnormal
    if T > 4:
        x[4] *= np.float32(5e37)
    if T > 5:
        x[5, 0, 3], x[5, 1, D - 1], x[5, 2, 40] = np.nan, np.inf, -np.inf
    if T > 6:
        x[6] *= np.exp(rng.uniform(-30, 30, (H, D))).astype(np.float32)  # far apart
    return torch.from_numpy(x).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kind", ["bf16", "q8", "q4"])
@pytest.mark.parametrize("D,page,T", [(64, 16, 1), (128, 16, 9), (256, 32, 40), (128, 64, 333), (64, 256, 257)])
def test_values_against_the_definition(gpu_ctx, kind, dtype, D, page, T):
    H = 3
    n_pages = -(-T // page) + 2
    c = make(gpu_ctx, kind, D, page, n_pages, H)
    k, v = hard_rows(T, H, D, dtype, 1), hard_rows(T, H, D, dtype, 2)
    slots = torch.randperm(n_pages * page, generator=torch.Generator().manual_seed(T))[:T].to(torch.int32)
    c.write(k.cuda(), v.cuda(), slots.cuda())
    for out in (torch.float32, torch.bfloat16):
        got = c.read(slots.cuda(), dtype=out)
        for x, y in zip((k, v), got):
            assert same(y.cpu(), torch.from_numpy(held(x.float().numpy(), kind)).to(out))
    gpu_ctx.synchronize()


@pytest.mark.parametrize("kind", ["bf16", "q8", "q4"])
def test_step_bound(gpu_ctx, kind):
    """A held value is at most half a step from what was written: bf16 2^-8 of it, q8 d / 2, q4 d / 2 with d rounded to bf16 (2^-8 of 7 steps for the largest)."""
    x = torch.randn((50, 3, 128), generator=torch.Generator().manual_seed(3))
    c = make(gpu_ctx, kind, 128)
    slots = torch.arange(50, dtype=torch.int32, device="cuda")
    c.write(x.cuda(), x.cuda(), slots)
    for y in c.read(slots, dtype=torch.float32):
        err = (y.cpu().double() - x.double()).abs()
        if kind == "bf16":
            assert (err <= 2.0 ** -8 * x.abs()).all()
        else:
            n, top = (128, 127) if kind == "q8" else (32, 7)
            d = x.double().reshape(50, 3, -1, n).abs().amax(-1, keepdim=True) / top
            assert (err.reshape(50, 3, -1, n) <= d * (0.5 + (top + 1) * (2.0 ** -8 if kind == "q4" else 2.0 ** -23))).all()


@pytest.mark.parametrize("kind", ["bf16", "q8", "q4"])
def test_only_the_named_rows_change(gpu_ctx, kind):
    H, D = 3, 128
    c = make(gpu_ctx, kind, D, 16, 9, H)
    every = torch.arange(144, dtype=torch.int32, device="cuda")
    old = torch.randn((144, H, D), generator=torch.Generator().manual_seed(5)).cuda()
    c.write(old, -old, every)
    before = [t.clone() for t in c.read(every, dtype=torch.float32)]
    new = torch.randn((6, H, D), generator=torch.Generator().manual_seed(6)).cuda()
    slots = torch.tensor([17, -1, 143, -5, 0, -2147483648], dtype=torch.int32, device="cuda")
    c.write(new, new * 2, slots)
    after = c.read(every, dtype=torch.float32)
    gpu_ctx.synchronize()
    for y, b, x in zip(after, before, (new, new * 2)):
        want = b.clone()
        for i, s in enumerate(slots.tolist()):
            if s >= 0:
                want[s] = torch.from_numpy(held(x[i].cpu().numpy(), kind)).cuda()
        assert torch.equal(y, want)
    k, v = c.read(slots, dtype=torch.bfloat16)
    assert not k[[1, 3, 5]].any() and not v[[1, 3, 5]].any() and k[0].any()


def test_slots_that_are_not_there_are_reported(gpu_ctx):
    c = make(gpu_ctx, "q8", 64, 16, 2, 3)
    x = torch.ones((3, 3, 64), device="cuda")
    c.write(x, x, torch.tensor([0, 31, 5], dtype=torch.int32, device="cuda"))
    gpu_ctx.synchronize()
    c.write(2 * x, 2 * x, torch.tensor([1, 32, 6], dtype=torch.int32, device="cuda"))
    with pytest.raises(B200MoeError, match="code 4"):
        gpu_ctx.synchronize()
    k, _ = c.read(torch.tensor([0, 1, 31, 6, 2147483647], dtype=torch.int32, device="cuda"), dtype=torch.float32)
    with pytest.raises(B200MoeError, match="code 4"):
        gpu_ctx.synchronize()
    assert [float(r.float().mean()) for r in k] == [1.0, 2.0, 1.0, 2.0, 0.0]
    gpu_ctx.synchronize()                               # reported once


@pytest.mark.parametrize("kind", ["bf16", "q8", "q4"])
def test_strided_unaligned_and_given_outputs(gpu_ctx, kind):
    T, H, D = 21, 3, 64
    g = torch.Generator().manual_seed(7)
    qkv = torch.randn((T, 4 + 2 * H, D), generator=g).to(torch.bfloat16).cuda()
    slots = torch.arange(T, dtype=torch.int32, device="cuda") + 5
    a, b = make(gpu_ctx, kind, D), make(gpu_ctx, kind, D)
    a.write(qkv[:, 4:4 + H].contiguous(), qkv[:, 4 + H:].contiguous(), slots)
    b.write(qkv[:, 4:4 + H], qkv[:, 4 + H:], slots)
    odd = torch.empty(T * H * D + 1, dtype=torch.bfloat16, device="cuda")[1:].view(T, H, D)
    odd.copy_(qkv[:, 4:4 + H])
    c = make(gpu_ctx, kind, D)
    c.write(odd, qkv[:, 4 + H:], slots)
    for n in ("k", "v") + (() if kind == "bf16" else ("k_scale", "v_scale")):
        assert torch.equal(getattr(a, n), getattr(b, n)) and torch.equal(getattr(a, n), getattr(c, n))
    want = a.read(slots)
    wide = torch.zeros((T, 2 * H + 1, D), dtype=torch.bfloat16, device="cuda")
    a.read(slots, out=(wide[:, :H], wide[:, H + 1:]))
    assert torch.equal(wide[:, :H], want[0]) and torch.equal(wide[:, H + 1:], want[1]) and not wide[:, H].any()
    a.read(slots, out=(odd, wide[:, H + 1:]))
    assert torch.equal(odd, want[0])
    # heads before tokens
    k, v = (torch.empty((H, T, D), dtype=torch.bfloat16, device="cuda").transpose(0, 1) for _ in range(2))
    a.read(slots, out=(k, v))
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


def test_one_row_for_all_heads_and_empty_calls(gpu_ctx):
    c = make(gpu_ctx, "q8", 128)
    x = torch.randn((4, 1, 128), device="cuda")
    slots = torch.arange(4, dtype=torch.int32, device="cuda")
    c.write(x.expand(4, 3, 128), x.expand(4, 3, 128), slots)
    k, v = c.read(slots, dtype=torch.float32)
    assert torch.equal(k, v) and torch.equal(k[:, 0], k[:, 2])
    c.write(x[:0].expand(0, 3, 128), x[:0].expand(0, 3, 128), slots[:0])
    assert c.read(slots[:0])[0].shape == (0, 3, 128)
    with pytest.raises(TypeError):
        c.write(x.expand(4, 3, 128), x.expand(4, 3, 128).bfloat16(), slots)
    with pytest.raises(ValueError):
        c.write(x.expand(4, 3, 128), x.expand(4, 3, 128), slots.long())
    with pytest.raises(ValueError):
        c.write(x.expand(4, 3, 128), x.expand(4, 3, 128), slots[:3])
    with pytest.raises(B200MoeError):
        c.write(x, x, slots)                            # one head for three
    with pytest.raises(ValueError):
        KvCache(gpu_ctx, kind="q8", n_pages=1, page_size=24, n_head_kv=1, head_dim=64)
    with pytest.raises(ValueError):
        KvCache(gpu_ctx, kind="q5", n_pages=1, page_size=16, n_head_kv=1, head_dim=64)


@pytest.mark.parametrize("kind", ["bf16", "q8"])
def test_offsets_beyond_32_bits(gpu_ctx, kind):
    D, H, page = 256, 8, 256
    n_pages = (5 << 30) // (D * H * page * (2 if kind == "bf16" else 1))
    c = make(gpu_ctx, kind, D, page, n_pages, H)
    assert c.k.numel() > (4 << 30)
    last = n_pages * page - 1
    slots = torch.tensor([0, last, last // 2, 1], dtype=torch.int32, device="cuda")
    x = torch.randn((4, H, D), generator=torch.Generator().manual_seed(1))
    c.write(x.cuda(), -x.cuda(), slots)
    k, v = c.read(slots, dtype=torch.float32)
    want = torch.from_numpy(held(x.numpy(), kind))
    assert torch.equal(k.cpu(), want) and torch.equal(v.cpu(), -want)
    row = D * (2 if kind == "bf16" else 1)
    rows = set((c.k.view(-1, row) != 0).any(-1).nonzero().flatten().tolist())
    assert rows == {((s // page) * H + h) * page + s % page for s in slots.tolist() for h in range(H)}
