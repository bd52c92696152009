"""Attention over the paged cache (b200moe_attention) against softmax in 64 bits over the values that the cache holds (b200moe_kv_read).

Tolerance, per output: half a step of the output's type relative to the value (bf16 2^-8, fp32 2^-24), plus the weights' errors times
sum_j p_j |v_j|:  2 ds for the scores' errors ds (they act on numerator and sum alike), w for the weights' own rounding (to f16, 2^-11, for bf16
queries; 2^-21 with the exponential's 2 ulp for fp32 ones) and 2^-24 for each of about L / 64 + 64 additions.  ds = (D / 16 + 8) 2^-23 times the
largest scale sum |q| |k| of the row: a run of D / 16 instructions that drop at most the accumulator's last bit each, and a few roundings
of the factors around it.  For bf16 queries the output accumulator, too, drops a last bit in each of its L / 64 steps: 2^-23 there.

f16 has a smallest step, too.  A weight times its key's scale is an f16 number below 2^14 (2^15 in the kernel for many rows), rounded by at most
2^-25; the largest weight of a row times the largest scale comes out at 2^13 or more there (2^6 or more), so a key's error is at most 2^-38
(2^-31) of the largest |v|, and with a second term for fp32 queries 2^-38 as well: L times that on top.  It shows where an output is
made of weights that small alone: a value of zero at the key that has nearly all the weight."""
import math

import numpy as np
import pytest
import torch

from edge0_b200.capi import B200MoeError
from edge0_b200.kv_cache import KvCache

pytestmark = pytest.mark.gpu


class Batch:
    """Sequences with random keys and values behind a prefix, and what their new tokens' attention should be."""

    def __init__(self, ctx, kind, lens, new=None, prefix=0, n_head=8, n_kv=2, D=128, page=16, dtype=torch.bfloat16, seed=0, spare=0, loud=1.0, wide_table=0):
        g = torch.Generator().manual_seed(seed)
        self.ctx, self.lens, self.new, self.prefix, self.dtype = ctx, list(lens), list(new or [1] * len(lens)), prefix, dtype
        self.n_head, self.n_kv, self.D, self.page = n_head, n_kv, D, page
        per = max(1, max(-(-n // page) for n in self.lens)) + wide_table
        per_prefix = -(-prefix // page)
        n_pages = per * len(self.lens) + per_prefix + spare
        order = torch.randperm(n_pages, generator=g).to(torch.int32)
        self.pages = order[:per * len(self.lens)].reshape(len(self.lens), per).cuda()
        self.prefix_pages = order[per * len(self.lens):per * len(self.lens) + per_prefix].cuda()
        self.cache = KvCache(ctx, kind=kind, n_pages=n_pages, page_size=page, n_head_kv=n_kv, head_dim=D)
        shape = (n_pages * page, n_kv, D)
        self.k, self.v = (torch.randn(shape, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
        self.k[..., 3] *= 4
        self.slots = torch.arange(n_pages * page, dtype=torch.int32, device="cuda")
        self.cache.write(self.k, self.v, self.slots)
        self.kv_len = torch.tensor(self.lens, dtype=torch.int32, device="cuda")
        self.q_start = torch.tensor([0] + list(np.cumsum(self.new)), dtype=torch.int32, device="cuda")
        self.T = sum(self.new)
        self.q = (torch.randn((self.T, n_head, D), generator=g) * loud).to(dtype).cuda()

    def held(self):
        return [t.double().view(-1, self.page, self.n_kv, self.D) for t in self.cache.read(self.slots, dtype=torch.float32)]

    def expected(self, scale=None, poisoned=None):
        """(out, lse, tolerance) in float64; what a token must not see is not looked at."""
        scale = self.D ** -0.5 if scale is None else scale
        k, v = self.held()
        G = self.n_head // self.n_kv
        out = torch.zeros((self.T, self.n_head, self.D), dtype=torch.float64, device="cuda")
        lse = torch.full((self.T, self.n_head), -math.inf, dtype=torch.float64, device="cuda")
        tol = torch.zeros_like(out)
        t = 0
        for b, (n, length) in enumerate(zip(self.new, self.lens)):
            kk, vv = (torch.cat([x[self.prefix_pages.long()].flatten(0, 1)[:self.prefix], x[self.pages[b].long()].flatten(0, 1)[:length]]) for x in (k, v))
            for i in range(n):
                seen = self.prefix + max(0, length - n + i + 1)
                if seen:
                    a, w = (x[:seen].repeat_interleave(G, 1) for x in (kk, vv))
                    q = self.q[t].double()
                    s = torch.einsum("hd,khd->hk", q, a) * scale
                    p = torch.softmax(s, -1)
                    lse[t] = torch.logsumexp(s, -1)
                    out[t] = torch.einsum("hk,khd->hd", p, w)
                    ds = (self.D / 16 + 8) * 2.0 ** -23 * (torch.einsum("hd,khd->hk", q.abs(), a.abs()).amax(-1) * abs(scale) + lse[t].abs())
                    f32 = self.dtype == torch.float32
                    own = 2.0 ** -21 if f32 else 2.0 ** -11
                    weight = 2 * ds + own + (seen / 64 + 64) * (2.0 ** -24 if f32 else 2.0 ** -23)
                    tol[t] = weight[:, None] * torch.einsum("hk,khd->hd", p, w.abs()) + (2.0 ** -24 if f32 else 2.0 ** -8) * out[t].abs() + 1e-30
                    tol[t] += seen * (2.0 ** -38 if f32 else 2.0 ** -31) * w.abs().amax(dim=(0, 2))[:, None]
                t += 1
        return out, lse, tol

    def call(self, **kw):
        a = dict(max_kv_len=max(self.lens), q_start=self.q_start, max_new=max(self.new), prefix_pages=self.prefix_pages, prefix_len=self.prefix)
        a.update(kw)
        return self.cache.attend(a.pop("q", self.q), a.pop("kv_len", self.kv_len), a.pop("pages", self.pages), **a)

    def check(self, **kw):
        lse = torch.full((self.T, self.n_head), 7.0, device="cuda")
        out = self.call(lse=lse, **kw)
        self.ctx.synchronize()
        want, want_lse, tol = self.expected(kw.get("scale"))
        err = (out.double() - want).abs()
        assert (err <= tol).all(), (float((err / tol).max()), int((err > tol).sum()), err.numel())
        assert torch.equal(torch.isinf(lse), torch.isinf(want_lse))
        fin = torch.isfinite(want_lse)
        assert ((lse.double() - want_lse).abs()[fin] <= 2e-5 * (1 + want_lse.abs()[fin])).all()
        return out


KINDS = ["bf16", "q8", "q4"]
DTYPES = [torch.bfloat16, torch.float32]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_ragged_decode(gpu_ctx, kind, D, dtype):
    Batch(gpu_ctx, kind, [1, 15, 16, 17, 127, 128, 129, 300, 31], D=D, dtype=dtype, seed=D).check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n_head,n_kv", [(1, 1), (3, 3), (7, 1), (12, 4), (16, 1), (17, 1), (40, 2), (66, 2)])
def test_head_layouts(gpu_ctx, kind, n_head, n_kv, dtype):
    b = Batch(gpu_ctx, kind, [40, 3, 133], n_head=n_head, n_kv=n_kv, dtype=dtype, seed=n_head, prefix=37)
    b.check()


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("kind", KINDS)
def test_pages_that_end_inside_a_tile(gpu_ctx, kind, page):
    for length in (page - 1, page, page + 1, 3 * page + 5):
        Batch(gpu_ctx, kind, [length, 1], page=page, prefix=length, seed=length).check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_shared_prefix(gpu_ctx, kind, D, dtype):
    Batch(gpu_ctx, kind, [5, 90, 1, 44], prefix=1000, n_head=160, n_kv=40, D=D, dtype=dtype, seed=1).check()
    Batch(gpu_ctx, kind, [5] * 33, prefix=333, n_head=20, n_kv=10, D=D, dtype=dtype, seed=2).check()
    Batch(gpu_ctx, kind, [5] * 33, prefix=1777, D=D, dtype=dtype, seed=2).check()
    Batch(gpu_ctx, kind, [20], prefix=1, D=D, dtype=dtype, seed=3).check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_short_prefix_and_few_blocks(gpu_ctx, kind, D, dtype):
    """Prefixes that are walked with the own keys, in one block and in clusters of two to sixteen that join themselves."""
    Batch(gpu_ctx, kind, [100, 7], prefix=37, D=D, dtype=dtype, seed=1).check()
    Batch(gpu_ctx, kind, [700, 20, 333], prefix=16, D=D, dtype=dtype, seed=2).check()
    Batch(gpu_ctx, kind, [3], prefix=2500, D=D, dtype=dtype, seed=3).check()
    Batch(gpu_ctx, kind, [2100, 0], prefix=101, new=[3, 2], n_head=6, n_kv=1, D=D, dtype=dtype, seed=4, page=32).check()
    Batch(gpu_ctx, kind, [300] * 9, n_head=16, n_kv=8, D=D, dtype=dtype, seed=5).check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new,lens,prefix", [
    ([3], [3], 0),                          # a whole prompt
    ([2, 5, 1, 4], [2, 90, 7, 131], 0),
    ([70], [200], 50),
    ([33, 1, 64], [40, 300, 64], 129),
    ([4, 4], [2, 0], 0),                    # fewer positions than new tokens: the first see nothing
    ([4, 4], [2, 0], 20),
    ([0, 3, 0], [50, 9, 0], 0),             # sequences without new tokens
])
def test_several_new_tokens(gpu_ctx, kind, new, lens, prefix, dtype):
    for n_head, n_kv in ((8, 2), (5, 5)):
        Batch(gpu_ctx, kind, lens, new=new, prefix=prefix, n_head=n_head, n_kv=n_kv, dtype=dtype, seed=sum(new)).check()


@pytest.mark.parametrize("kind", KINDS)
def test_empty_sequences(gpu_ctx, kind):
    out = Batch(gpu_ctx, kind, [0, 5, 0, 33]).check(max_kv_len=33)
    assert not out[0].any() and not out[2].any()
    Batch(gpu_ctx, kind, [0, 0], prefix=40).check(max_kv_len=0)
    out = Batch(gpu_ctx, kind, [0, 0]).check(max_kv_len=0)
    assert not out.any()
    out = Batch(gpu_ctx, kind, [0, 0], wide_table=60).check(max_kv_len=900)
    assert not out.any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
def test_long(gpu_ctx, kind, dtype):
    Batch(gpu_ctx, kind, [20011, 1], page=64, dtype=dtype, n_head=8, n_kv=1, wide_table=3).check()
    Batch(gpu_ctx, kind, [700, 2], page=64, dtype=dtype, prefix=9001, n_head=8, n_kv=1).check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
def test_bounds_wider_than_the_lengths_and_the_split_change_nothing(gpu_ctx, kind, dtype):
    b = Batch(gpu_ctx, kind, [9, 200, 64], dtype=dtype, wide_table=70)
    b.check(max_kv_len=None)
    b.check(max_kv_len=201)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("loud", [1e-20, 1e-3, 30.0])
def test_query_sizes(gpu_ctx, kind, loud):
    for dtype in DTYPES:
        Batch(gpu_ctx, kind, [50, 260], dtype=dtype, loud=loud, seed=4).check()


@pytest.mark.parametrize("scale", [0.0, -0.1, 1.0])
def test_scales(gpu_ctx, scale):
    for kind in KINDS:
        Batch(gpu_ctx, kind, [50, 260], n_head=4, seed=4).check(scale=scale)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_values_of_very_different_sizes(gpu_ctx, kind, dtype):
    """Rows whose values are 10^12 apart: the weights' common factor follows the largest that was seen."""
    b = Batch(gpu_ctx, kind, [400, 37], dtype=dtype)
    size = torch.exp(torch.rand(b.v.shape[0], 1, 1, generator=torch.Generator().manual_seed(3)) * 28 - 14).cuda()
    b.cache.write(b.k, (b.v.float() * size).to(torch.bfloat16), b.slots)
    b.check()
    b.cache.write(b.k, b.v * 1e-30, b.slots)
    b.check()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new", [None, [9, 3]])
@pytest.mark.parametrize("what", ["nan", "inf", "bytes"])
def test_what_lies_out_of_reach_has_no_influence(gpu_ctx, kind, new, what):
    """Everything that no token sees - the rest of the last pages, other pages, and for a token the new ones behind it - is not a number, or any bytes."""
    b = Batch(gpu_ctx, kind, [21, 130], new=new, prefix=19, spare=3)
    clean = b.check()
    used = torch.zeros(b.slots.numel(), dtype=torch.bool, device="cuda").view(-1, b.page)
    for s, n in enumerate(b.lens):
        for i in range(n):
            used[b.pages[s, i // b.page].long(), i % b.page] = True
    for i in range(b.prefix):
        used[b.prefix_pages[i // b.page].long(), i % b.page] = True
    free = b.slots[~used.flatten()].contiguous()
    if what == "bytes":
        for name in ("k", "v", "k_scale", "v_scale"):
            t = getattr(b.cache, name)
            if t is not None:
                rows = t.view(-1, b.n_kv, b.page, t.numel() // (used.numel() * b.n_kv))
                rows.transpose(1, 2)[~used] = 255
    else:
        bad = torch.full((free.numel(), b.n_kv, b.D), float(what), dtype=torch.bfloat16, device="cuda")
        b.cache.write(bad, bad, free)
    assert torch.equal(b.call(), clean)
    if new:
        # the last new token's own rows: nothing for those before it, everything for itself
        last = [b.pages[s, (n - 1) // b.page] * b.page + (n - 1) % b.page for s, n in enumerate(b.lens)]
        x = torch.full((2, b.n_kv, b.D), float("nan" if what == "bytes" else what), dtype=torch.bfloat16, device="cuda")
        b.cache.write(x, x, torch.stack(last).to(torch.int32))
        out = b.call()
        ends = [new[0] - 1, sum(new) - 1]
        others = [t for t in range(b.T) if t not in ends]
        assert torch.equal(out[others], clean[others])
        assert not torch.isfinite(out[ends]).any()
    b.ctx.synchronize()


@pytest.mark.parametrize("kind", KINDS)
def test_nan_within_reach_is_seen(gpu_ctx, kind):
    b = Batch(gpu_ctx, kind, [300, 40], prefix=16)
    clean = b.call()
    x = torch.zeros((1, b.n_kv, b.D), dtype=torch.bfloat16, device="cuda")
    x[0, 1, 5] = float("nan")
    b.cache.write(torch.zeros_like(x), x, (b.pages[0, 3] * b.page + 2).to(torch.int32).reshape(1))
    out = b.call()
    G = b.n_head // b.n_kv
    cols = {"bf16": slice(5, 6), "q8": slice(0, b.D), "q4": slice(0, 32)}[kind]
    bad = torch.zeros(out.shape, dtype=torch.bool, device="cuda")
    bad[0, G:, cols] = True
    assert torch.equal(torch.isnan(out), bad)
    assert torch.equal(out[1], clean[1])
    b.cache.write(x, torch.zeros_like(x), (b.prefix_pages[0] * b.page).to(torch.int32).reshape(1))
    assert torch.isnan(b.call()[:, G:]).all() and torch.isfinite(b.call()[:, :G]).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("what", ["inf", "nan"])
def test_the_other_columns_of_a_row_with_an_infinity(gpu_ctx, kind, what):
    """A value that is not finite spoils outputs of its head only; in a BF16 cache, where a row has no scale, its own column alone (or, where some token
    does not see the key, the head), and never another value's share."""
    for n_head, new in ((8, None), (256, None), (8, [40, 40])):
        b = Batch(gpu_ctx, kind, [300, 90], new=new, n_head=n_head, n_kv=2, prefix=64)
        clean, _, tol = b.expected()
        G = n_head // 2
        x = b.v[(b.prefix_pages[1] * b.page + 2).long()][None].clone()
        x[0, 1, 5] = float(what)
        b.cache.write(b.k[(b.prefix_pages[1] * b.page + 2).long()][None].contiguous(), x, (b.prefix_pages[1] * b.page + 2).to(torch.int32).reshape(1))
        out = b.call()
        assert ((out[:, :G].double() - clean[:, :G]).abs() <= tol[:, :G]).all()
        assert not torch.isfinite(out[:, G:, 5]).any()
        rest = torch.ones(b.D, dtype=torch.bool, device="cuda")
        rest[{"bf16": slice(5, 6), "q8": slice(0, b.D), "q4": slice(0, 32)}[kind]] = False
        got, want, bound = out[:, G:, rest].double(), clean[:, G:, rest], tol[:, G:, rest]
        assert ((got - want).abs() <= bound).logical_or(torch.isnan(got)).all()
        if new is None:
            assert torch.isfinite(got).all()
    gpu_ctx.synchronize()


def test_many_rows_behind_the_last_sequence(gpu_ctx):
    for prefix in (0, 3000):
        b = Batch(gpu_ctx, "q4", [130, 200], new=[20, 31], prefix=prefix)
        want, _, tol = b.expected()
        q = torch.cat([b.q, torch.full((9, b.n_head, b.D), float("nan"), dtype=b.dtype, device="cuda")])
        out = torch.full_like(q, 3.0)
        b.call(q=q, out=out)
        assert ((out[:51].double() - want).abs() <= tol).all() and (out[51:] == 3).all()
        out.fill_(3.0)
        b.call(q=q, out=out, kv_len=torch.tensor([130, 201], dtype=torch.int32, device="cuda"))
        with pytest.raises(B200MoeError, match="code 5"):
            gpu_ctx.synchronize()
        assert ((out[:20].double() - want[:20]).abs() <= tol[:20]).all() and (out[20:] == 3).all()


def test_rows_behind_the_last_sequence_and_bad_lengths(gpu_ctx):
    b = Batch(gpu_ctx, "q8", [30, 200], new=[2, 3], prefix=50)
    b.check()
    want, _, tol = b.expected()
    near = lambda x, y, bound: bool(((x.double() - y).abs() <= bound).all())
    q = torch.cat([b.q, torch.full((7, b.n_head, b.D), float("nan"), dtype=b.dtype, device="cuda")])
    out = torch.full_like(q, 3.0)
    lse = torch.full(q.shape[:2], 9.0, device="cuda")
    b.call(q=q, out=out, lse=lse)
    assert near(out[:5], want, tol) and (out[5:] == 3).all() and (lse[5:] == 9).all() and (lse[:5] != 9).all()
    gpu_ctx.synchronize()
    # without q_start, more rows than sequences
    one = Batch(gpu_ctx, "q8", [30, 200], prefix=50)
    want1, _, tol1 = one.expected()
    q1 = torch.cat([one.q, one.q])
    out1 = torch.full_like(q1, 3.0)
    one.call(q=q1, out=out1, q_start=None)
    assert near(out1[:2], want1, tol1) and (out1[2:] == 3).all()
    # a length beyond the bound, below zero, too many new tokens, a table of starts that goes back: reported, those rows left alone
    for kw, left in ((dict(kv_len=torch.tensor([30, 201], dtype=torch.int32, device="cuda")), [2, 3, 4]),
                     (dict(kv_len=torch.tensor([-1, 200], dtype=torch.int32, device="cuda")), [0, 1]),
                     (dict(max_new=2), [2, 3, 4]),
                     (dict(q_start=torch.tensor([0, 2, 9], dtype=torch.int32, device="cuda")), [2, 3, 4])):
        out.fill_(3.0)
        b.call(q=b.q, out=out[:5], **kw)
        with pytest.raises(B200MoeError, match="code 5"):
            gpu_ctx.synchronize()
        for t in range(5):
            assert (out[t] == 3).all() if t in left else near(out[t], want[t], tol[t])
    gpu_ctx.synchronize()


@pytest.mark.parametrize("kind", KINDS)
def test_pages_that_are_not_there_are_reported(gpu_ctx, kind):
    b = Batch(gpu_ctx, kind, [64, 64])
    want = b.check()
    _, _, tol = b.expected()
    for page in (-1, b.cache.n_pages, 2 ** 31 - 1):
        pages = b.pages.clone()
        pages[0, 1] = page
        out = b.call(pages=pages)
        with pytest.raises(B200MoeError, match="code 4"):
            gpu_ctx.synchronize()
        assert torch.equal(out[1], want[1]) and torch.isfinite(out[0]).all() and not torch.equal(out[0], want[0])
    # entries behind a sequence's length are not looked at
    pages = torch.cat([b.pages, torch.full((2, 3), -7, dtype=torch.int32, device="cuda")], dim=1)
    assert ((b.call(pages=pages.contiguous(), max_kv_len=100).double() - want.double()).abs() <= 2 * tol).all()
    gpu_ctx.synchronize()


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(gpu_ctx, dtype):
    b = Batch(gpu_ctx, "q8", [70, 9, 133], n_head=6, n_kv=2, dtype=dtype)
    want = b.check()
    wide = torch.randn((3, 6 + 4, 128), device="cuda").to(dtype)
    wide[:, :6] = b.q
    keep = wide.clone()
    assert torch.equal(b.call(q=wide[:, :6]), want)
    out = torch.full((6, 3, 130), 2.0, device="cuda").to(dtype)
    b.call(q=wide[:, :6], out=out[:, :, 1:129].transpose(0, 1))
    assert torch.equal(out[:, :, 1:129].transpose(0, 1), want) and (out[:, :, 0] == 2).all() and (out[:, :, 129] == 2).all()
    assert torch.equal(wide, keep)
    # the result over the queries
    b.call(q=wide[:, :6], out=wide[:, :6])
    assert torch.equal(wide[:, :6], want) and torch.equal(wide[:, 6:], keep[:, 6:])


def test_graph_replayed_with_other_lengths_beside_another(gpu_ctx):
    """Two captured calls with workspaces of their own, replayed on two streams at once; lengths, tables and queries change between replays."""
    a = Batch(gpu_ctx, "q8", [500, 77, 3], prefix=300, seed=1)
    b = Batch(gpu_ctx, "bf16", [40, 900], prefix=64, seed=2, new=[5, 2])
    graphs, outs = [], []
    for x, bound in ((a, 600), (b, 1000)):
        x.pages = torch.cat([x.pages, torch.zeros((len(x.lens), 40), dtype=torch.int32, device="cuda")], dim=1).contiguous()
        out = torch.zeros_like(x.q)
        x.call(out=out, max_kv_len=bound)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            x.call(out=out, max_kv_len=bound)
        graphs.append(g)
        outs.append(out)
    streams = [torch.cuda.Stream() for _ in graphs]
    for step in range(6):
        a.lens = [[500, 77, 3], [1, 2, 499], [0, 400, 64], [128, 129, 127], [500, 500, 500], [16, 16, 16]][step]
        a.lens = [min(n, 512) for n in a.lens]
        a.kv_len.copy_(torch.tensor(a.lens, dtype=torch.int32))
        a.pages[:, :32] = a.pages[:, :32].roll(1, 0)
        b.q.copy_(torch.randn(b.q.shape, generator=torch.Generator().manual_seed(step)).to(b.dtype))
        for o in outs:
            o.fill_(5.0)
        torch.cuda.synchronize()
        for _ in range(3):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for x, o in zip((a, b), outs):
            want, _, tol = x.expected()
            assert ((o.double() - want).abs() <= tol).all()
    gpu_ctx.synchronize()


def test_same_bits_every_time(gpu_ctx):
    b = Batch(gpu_ctx, "q4", [3000, 77, 900], prefix=2000, page=64)
    first = b.call()
    for _ in range(5):
        assert torch.equal(b.call(), first)


def test_rope_write_attend_as_a_decoder_layer_does(gpu_ctx):
    """A prompt in two chunks, then three steps of one token: rotary positions, the cache, attention, against the same in 64 bits over held values."""
    H, Hk, D, page = 8, 2, 64, 32
    g = torch.Generator().manual_seed(11)
    lens = [50, 23]
    cache = KvCache(gpu_ctx, kind="q8", n_pages=8, page_size=page, n_head_kv=Hk, head_dim=D)
    pages = torch.tensor([[5, 2, 0], [7, 1, 3]], dtype=torch.int32, device="cuda")
    have = [0, 0]
    steps = [[30, 20], [20, 3], [1, 1], [1, 1], [1, 1]]
    for new in steps:
        T = sum(new)
        qkv = torch.randn((T, H + 2 * Hk, D), generator=g).to(torch.bfloat16).cuda()
        where = [(b, have[b] + i) for b, n in enumerate(new) for i in range(n)]
        pos = torch.tensor([i for _, i in where], dtype=torch.int32, device="cuda")
        slots = torch.tensor([int(pages[b, i // page]) * page + i % page for b, i in where], dtype=torch.int32, device="cuda")
        turned = gpu_ctx.rope(qkv[:, :H + Hk], pos, base=1e4)
        cache.write(turned[:, H:], qkv[:, H + Hk:], slots)
        have = [h + n for h, n in zip(have, new)]
        out = cache.attend(turned[:, :H], torch.tensor(have, dtype=torch.int32, device="cuda"), pages,
                           q_start=torch.tensor([0, new[0], T], dtype=torch.int32, device="cuda"), max_new=max(new))
        gpu_ctx.synchronize()
        # the formulas: turn, hold, attend
        freq = 1e4 ** (-torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D)
        w = pos.double()[:, None, None] * freq
        x = qkv[:, :H + Hk].double()
        ref = torch.cat([x[..., :D // 2] * w.cos() - x[..., D // 2:] * w.sin(), x[..., :D // 2] * w.sin() + x[..., D // 2:] * w.cos()], -1)
        assert ((turned.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -20).all()
        k, v = (t.double() for t in cache.read(torch.arange(8 * page, dtype=torch.int32, device="cuda"), dtype=torch.float32))
        step = turned[:, H:].double().abs().amax(-1, keepdim=True) / 127
        assert ((k[slots.long()] - turned[:, H:].double()).abs() <= step * 0.5001).all()
        for t, (b, i) in enumerate(where):
            rows = torch.tensor([int(pages[b, j // page]) * page + j % page for j in range(i + 1)], device="cuda")
            a, u = (z[rows].repeat_interleave(H // Hk, 1) for z in (k, v))
            p = torch.softmax(torch.einsum("hd,khd->hk", turned[t, :H].double(), a) / math.sqrt(D), -1)
            want = torch.einsum("hk,khd->hd", p, u)
            err = (out[t].double() - want).abs()
            assert (err <= 2.0 ** -8 * want.abs() + 2.0 ** -10 * torch.einsum("hk,khd->hd", p, u.abs())).all()


def test_refusals(gpu_ctx):
    b = Batch(gpu_ctx, "q8", [30, 200], prefix=500, n_head=66, n_kv=66)
    with pytest.raises(B200MoeError):
        b.call(max_kv_len=300)
    with pytest.raises(ValueError):
        b.call(prefix_len=513)
    with pytest.raises(ValueError):
        b.call(prefix_pages=None)
    with pytest.raises(ValueError):
        b.call(pages=b.pages.long())
    with pytest.raises(ValueError):
        b.call(pages=b.pages[:1])
    with pytest.raises(ValueError):
        b.call(q_start=b.q_start[:2])
    with pytest.raises(ValueError):
        b.call(out=b.q[:1])
    with pytest.raises(TypeError):
        b.call(q=b.q.half())
    with pytest.raises(ValueError):
        b.call(q=b.q.cpu())
    with pytest.raises(ValueError):
        b.call(kv_len=b.kv_len.cpu())
    with pytest.raises(B200MoeError):
        b.call(q_start=None, max_new=2)
    with pytest.raises(B200MoeError):
        b.call(q=b.q[:, :65])
    with pytest.raises(B200MoeError):
        b.call(q=b.q[..., :64].contiguous())
    with pytest.raises(B200MoeError):
        b.call(workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    with pytest.raises(ValueError):
        b.call(lse=torch.empty(3, device="cuda"))
    gpu_ctx.synchronize()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_prefix_of_a_wide_batch(gpu_ctx, kind, D, dtype):
    """Prefixes too long to be walked by every sequence: few rows to a key/value head, and many, of which some are nobody's."""
    Batch(gpu_ctx, kind, [5, 90, 1, 44, 0], prefix=2077, n_head=40, n_kv=20, D=D, dtype=dtype, seed=1).check()
    Batch(gpu_ctx, kind, [5, 70, 1] * 11, prefix=5003, n_head=32, n_kv=8, D=D, dtype=dtype, seed=2, page=64).check()
    b = Batch(gpu_ctx, kind, [9, 33] * 20, new=[3, 2] * 20, prefix=1200, n_head=28, n_kv=14, D=D, dtype=dtype, seed=3, page=32)
    b.check()
    want, _, tol = b.expected()
    q = torch.cat([b.q, torch.full((7, b.n_head, D), float("nan"), dtype=dtype, device="cuda")])
    out = torch.full_like(q, 3.0)
    b.call(q=q, out=out)
    assert ((out[:b.T].double() - want).abs() <= tol).all() and (out[b.T:] == 3).all()
    b.ctx.synchronize()


def test_many_rows_replayed_on_two_streams(gpu_ctx):
    """Graphs of the tensor-memory kernels side by side, lengths and tables changed between replays."""
    cases = [Batch(gpu_ctx, kind, [300, 170], new=[40, 40], n_head=16, n_kv=2, prefix=prefix, seed=7) for kind, prefix in (("bf16", 0), ("q8", 90), ("q4", 5000))]
    graphs, outs = [], []
    for x in cases:
        out = torch.zeros_like(x.q)
        x.call(out=out)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            x.call(out=out)
        graphs.append(g)
        outs.append(out)
    streams = [torch.cuda.Stream() for _ in graphs]
    for step, lens in enumerate(([300, 170], [41, 40], [0, 299], [256, 64])):
        for x, o in zip(cases, outs):
            x.lens = [min(n, 16 * x.pages.shape[1]) for n in lens]
            x.kv_len.copy_(torch.tensor(x.lens, dtype=torch.int32))
            x.q.copy_(torch.randn(x.q.shape, generator=torch.Generator().manual_seed(step)).to(x.dtype))
            o.fill_(5.0)
        torch.cuda.synchronize()
        for _ in range(3):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for x, o in zip(cases, outs):
            want, _, tol = x.expected()
            assert ((o.double() - want).abs() <= tol).all()
    gpu_ctx.synchronize()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("what", ["nan", "inf", "3e38"])
def test_many_rows_and_what_they_do_not_see(gpu_ctx, kind, what):
    """New tokens of a chunk see nothing of those behind them, be they infinite, not numbers or merely large."""
    b = Batch(gpu_ctx, kind, [250, 77, 64], new=[70, 77, 40], prefix=45)
    clean = b.check()
    tail = [3, 60, 40]    # of each sequence's new tokens are replaced
    slots = torch.cat([b.pages[s].repeat_interleave(b.page)[n - m:n] * b.page + torch.arange(n - m, n, device="cuda") % b.page
                       for s, (n, m) in enumerate(zip(b.lens, tail))]).to(torch.int32)
    x = torch.full((sum(tail), b.n_kv, b.D), float(what), dtype=torch.bfloat16, device="cuda")
    b.cache.write(x, x, slots)
    out = b.call()
    at = [0, 70, 147]
    before = torch.cat([torch.arange(a, a + n - m) for a, n, m in zip(at, b.new, tail)]).cuda()
    assert torch.equal(out[before], clean[before])
    if what != "3e38":
        behind = torch.tensor([t for t in range(b.T) if t not in set(before.tolist())], device="cuda")
        assert not torch.isfinite(out[behind]).any()
    b.ctx.synchronize()


@pytest.mark.parametrize("kind", ["q8", "q4"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [None, [80, 70]])
def test_queries_near_the_largest_number(gpu_ctx, kind, dtype, new):
    Batch(gpu_ctx, kind, [300, 90], new=new, dtype=dtype, loud=6e37).check(scale=128 ** -0.5 / 6e37)
