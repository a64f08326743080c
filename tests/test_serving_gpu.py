"""The serving operators on the GPU against their 64-bit forms (serving_ref.py,
where the tolerances are derived): rotary positions and their gradient, the
paged cache, attention over it, page copies, and a serving run of them all."""
import math

import pytest
import torch

import oracle
import serving_ref as ref

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32


def _gen(seed):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------------------------- rotary positions
@pytest.mark.parametrize("kw", [dict(), dict(scaling="linear", factor=4.0), dict(scaling="ntk", factor=8.0),
                                dict(scaling="yarn", factor=16.0, original_positions=4096), dict(base=500000.0)])
def test_rotary_table(fa, cuda, kw):
    n, r = 70000, 64
    table = fa.rotary_table(n, r, **kw).cpu()
    freqs, factor = fa.rotary_frequencies(r, **kw)
    angle = torch.arange(n, dtype=torch.float64)[:, None] * torch.tensor(freqs, dtype=torch.float64)
    want = factor * torch.stack((angle.cos(), angle.sin()), -1)
    # One rounding to FP32 (half a step of values up to factor), and 64-bit noise.
    assert float((table.double() - want).abs().max()) <= factor * (ref.EPS32 + 1e-10)


ROTARY = [  # B, H, S, D, rotary_dim
    (2, 3, 65, 128, 128),
    (1, 5, 130, 64, 64),
    (2, 2, 33, 96, 48),
    (1, 3, 17, 160, 160),
    (1, 2, 9, 256, 2),       # a single pair
    (3, 1, 20, 64, 22),      # no whole eights
    (1, 1, 1, 32, 32),
    (1, 40, 700, 128, 64),   # several heads a thread
]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("shape", ROTARY)
def test_rotary(fa, cuda, shape, dtype, interleaved):
    B, H, S, D, r = shape
    x = torch.randn(B, S, H, D, generator=_gen(1)).to(dtype).transpose(1, 2)
    pos = torch.randint(0, 5000, (B, S), generator=_gen(2)).int()
    table = fa.rotary_table(5000, r)
    y = fa.rotary(x.cuda(), table, pos.cuda(), interleaved=interleaved)
    assert y.is_contiguous() and y.dtype == dtype
    cos, sin = ref.angles(table.cpu(), pos[:, None])
    want, size = ref.rotate(x, cos, sin, interleaved)
    off = (y.cpu().double() - want).abs()
    assert bool((off <= ref.rotary_bound(want, size, dtype)).all()), float(off.max())
    assert torch.equal(y.cpu()[..., r:], x[..., r:])
    # positions shared by the batch, and the default ones
    one = fa.rotary(x.cuda(), table, pos[0].cuda(), interleaved=interleaved)
    assert torch.equal(one[0], y[0])
    count = fa.rotary(x.cuda(), table, interleaved=interleaved)
    assert torch.equal(count, fa.rotary(x.cuda(), table, torch.arange(S).int().cuda(), interleaved=interleaved))
    assert fa.status_query() == fa.OK


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_strides_and_in_place(fa, cuda, interleaved):
    """Views that start off a 16-byte boundary, odd strides, and out=x give the bytes of the plain call."""
    B, H, S, D = 2, 3, 19, 64
    table = fa.rotary_table(64, D)
    base = torch.randn(B, S, H, D + 3, generator=_gen(4)).half().cuda()
    x = base[..., 1:D + 1].transpose(1, 2)
    want = fa.rotary(x.contiguous(), table, interleaved=interleaved)
    assert torch.equal(fa.rotary(x, table, interleaved=interleaved), want)
    rest = base.clone()
    fa.rotary(x, table, interleaved=interleaved, out=x)
    assert torch.equal(x, want)
    assert torch.equal(base[..., 0], rest[..., 0]) and torch.equal(base[..., D + 1:], rest[..., D + 1:])
    flat = want.clone()
    fa.rotary(flat, table, interleaved=interleaved, out=flat)
    assert torch.equal(flat, fa.rotary(want, table, interleaved=interleaved))
    # every head the same memory
    e = x[:, :1].expand(B, H, S, D)
    assert torch.equal(fa.rotary(e, table), fa.rotary(e.contiguous(), table))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("dim,rot", [(32, 6), (64, 22), (96, 80), (128, 50), (128, 96), (160, 2), (256, 250)])
def test_rotary_dimensions_across_eights(fa, cuda, dim, rot, interleaved, dtype):
    """Aligned rows, unaligned rows and the rotation in place give the same bytes, and so does
    an append of the same rows."""
    B, H, S = 2, 5, 37
    table = fa.rotary_table(64, rot)
    base = torch.randn(B, S, H, dim + 1, generator=_gen(11)).to(dtype).cuda()
    off = base[..., 1:].transpose(1, 2)  # rows off a 16-byte boundary
    x = off.contiguous()
    want = fa.rotary(off, table, interleaved=interleaved)
    assert torch.equal(fa.rotary(x, table, interleaved=interleaved), want)
    pages = torch.arange(6, dtype=torch.int32, device="cuda").view(2, 3)
    pos = torch.arange(S, dtype=torch.int32, device="cuda").repeat(B)
    seq = torch.arange(B, dtype=torch.int32, device="cuda").repeat_interleave(S)
    got = []
    for rows in (x, off):
        cache = fa.PagedCache.empty(6, 16, H, dim)
        for t in (cache.k_codes, cache.k_scales, cache.v):
            t.zero_()
        r = rows.transpose(1, 2)
        r = r.reshape(B * S, H, dim) if rows is x else base.view(B * S, H, dim + 1)[..., 1:]
        q = fa.cache_append(cache, r, r, pages, pos, seq_ids=seq, Q=r, table=table, interleaved=interleaved)
        assert torch.equal(q, want.transpose(1, 2).reshape(B * S, H, dim))
        got.append((cache.k_codes, cache.k_scales, cache.v))
    assert all(torch.equal(a, b) for a, b in zip(*got))
    fa.rotary(x, table, interleaved=interleaved, out=x)
    assert torch.equal(x, want)


def test_outputs_that_cannot_be_written(fa, cuda):
    """out= with shared elements or half over the input is refused; out=x moves x's version on."""
    B, H, S, D = 2, 3, 8, 64
    table = fa.rotary_table(S, D)
    base = torch.randn(2 * B * H * S * D, generator=_gen(6)).half().cuda()
    x = base[:B * H * S * D].view(B, H, S, D)
    with pytest.raises(ValueError, match="share memory"):
        fa.rotary(x, table, out=x[:, :1].expand(B, H, S, D))
    with pytest.raises(ValueError, match="partly"):
        fa.rotary(x, table, out=base[D:D + B * H * S * D].view(B, H, S, D))
    beside = base[B * H * S * D:].view(B, H, S, D)
    assert torch.equal(fa.rotary(x, table, out=beside), fa.rotary(x, table))
    w = torch.randn(D, generator=_gen(7)).half().cuda().requires_grad_()
    loss = (x * w).sum()
    fa.rotary(x, table, out=x)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with pytest.raises(ValueError, match="no gradient"):
        fa.rotary_embedding(x, table.clone().requires_grad_())


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rot", [64, 30])
def test_rotary_gradient(fa, cuda, rot, interleaved):
    B, H, S, D = 2, 3, 21, 64
    table = fa.rotary_table(300, rot, scaling="yarn", factor=4.0, original_positions=128)
    pos = torch.randint(0, 300, (B, S), generator=_gen(7)).int()
    x = torch.randn(B, S, H, D, generator=_gen(5)).cuda().transpose(1, 2).requires_grad_()
    dy = torch.randn(B, H, S, D, generator=_gen(6))
    y = fa.rotary_embedding(x, table, pos.cuda(), interleaved=interleaved)
    (dx,) = torch.autograd.grad(y, x, dy.cuda())
    cos, sin = ref.angles(table.cpu(), pos[:, None])
    want, size = ref.rotate(dy, cos, -sin, interleaved)          # the formula
    assert bool(((dx.cpu().double() - want).abs() <= ref.rotary_bound(want, size, F32)).all())
    # Differences: y is linear in x, so <dy, R(x + t v) - R(x - t v)> / 2t = <dx, v> up to the rounding of y
    # (2^-23 of the products of every element), whatever t is.
    v = torch.randn(B, H, S, D, generator=_gen(8))
    f = [float((fa.rotary((x.detach().cpu() + t * v).cuda(), table, pos.cuda(), interleaved).cpu().double() *
                dy.double()).sum()) for t in (1.0, -1.0)]
    got = float((dx.cpu().double() * v.double()).sum())
    big = 2 * ref.EPS32 * float(((x.detach().cpu().abs() + v.abs()).double() * 2 * dy.abs().double()).sum()) * 4
    assert abs((f[0] - f[1]) / 2 - got) <= big
    # the gradient's gradient: dx = R^T dy is linear in dy
    w = dy.cuda().requires_grad_()
    (dx2,) = torch.autograd.grad(fa.rotary_embedding(x, table, pos.cuda(), interleaved), x, w, create_graph=True)
    assert torch.equal(dx2, dx)
    (dw,) = torch.autograd.grad(dx2, w, v.cuda())
    assert torch.equal(dw, fa.rotary(v.cuda(), table, pos.cuda(), interleaved))
    # a broadcast gradient (stride 0) is as its copy
    (d0,) = torch.autograd.grad(fa.rotary_embedding(x, table, pos.cuda(), interleaved).sum(), x)
    assert torch.equal(d0, fa.rotary(torch.ones(B, H, S, D).cuda(), table, pos.cuda(), interleaved, inverse=True))


def test_rotary_positions_out_of_range(fa, cuda):
    table = fa.rotary_table(8, 32)
    x = torch.randn(1, 2, 3, 64, generator=_gen(1)).half().cuda()
    y = fa.rotary(x, table, torch.tensor([7, 8, -1], dtype=torch.int32).cuda())
    assert fa.status_query() == fa.EINDEX
    assert b"position" in fa.lib().fp4attn_last_error()
    assert fa.status_query() == fa.OK
    assert bool((y[:, :, 1:] == 0).all())
    assert torch.equal(y[:, :, :1], fa.rotary(x[:, :, :1], table, torch.tensor([7], dtype=torch.int32).cuda()))


def test_rotary_gradient_under_capture(fa, cuda):
    """Forward and gradient captured (no eager graph of the leaf alive) and replayed on new inputs."""
    table = fa.rotary_table(64, 64)
    x = torch.randn(1, 2, 64, 64, generator=_gen(1)).cuda().requires_grad_()
    dy = torch.randn(1, 2, 64, 64, generator=_gen(2)).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # (autograd's own warm-up)
        torch.autograd.grad(fa.rotary_embedding(x, table), x, dy)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = fa.rotary_embedding(x, table)
        (dx,) = torch.autograd.grad(y, x, dy)
        y = y.detach()
    with torch.no_grad():
        x.copy_(torch.randn(1, 2, 64, 64, generator=_gen(3)))
        dy.copy_(torch.randn(1, 2, 64, 64, generator=_gen(4)))
    g.replay()
    assert torch.equal(y, fa.rotary(x.detach(), table))
    assert torch.equal(dx, fa.rotary(dy, table, inverse=True))


def test_rotary_under_capture(fa, cuda):
    table = fa.rotary_table(64, 64)
    x = torch.randn(1, 2, 64, 64, generator=_gen(1)).half().cuda()
    out = torch.empty_like(x)
    fa.rotary(x, table, out=out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        fa.rotary(x, table, out=out)
    x.copy_(torch.randn(1, 2, 64, 64, generator=_gen(2)).half())
    g.replay()
    assert torch.equal(out, fa.rotary(x, table))


# ------------------------------------------------------------------------------- the cache
def _blank(fa, pages, page, heads, dim, fill=True):
    """A cache whose unwritten places hold NaN values and scale bytes of 255 (NaN)."""
    c = fa.PagedCache.empty(pages, page, heads, dim)
    if fill:
        c.k_codes.fill_(0x77)
        c.k_scales.fill_(255)
        c.v.fill_(math.nan)
    return c


def _cpu(c):
    return c.k_codes.cpu(), c.k_scales.cpu(), c.v.cpu()


def _tables(seed, seqs, per_seq, pages):
    return torch.randperm(pages, generator=_gen(seed))[: seqs * per_seq].view(seqs, per_seq).int()


APPEND = [  # page, kv_heads, q_heads, D, rotary_dim, dtype, interleaved, ocp
    (64, 2, 4, 128, 128, F16, False, False),
    (16, 3, 3, 64, 64, F16, True, False),
    (32, 1, 5, 96, 48, F32, False, True),
    (128, 2, 2, 160, 22, F16, False, True),
    (16, 1, 2, 256, 256, F32, True, False),
    (64, 4, 4, 32, 0, F16, False, False),
]


def test_append_of_unaligned_rows(fa, cuda):
    """Rows off a 16-byte boundary and odd strides: the bytes of aligned rows."""
    for r, inter in ((64, False), (64, True), (0, False), (24, True)):
        base = torch.randn(9, 3, 64 + 5, generator=_gen(4)).half().cuda()
        x = base[:, :, 3:67]
        table = fa.rotary_table(32, r) if r else None
        got = []
        for t in (x, x.contiguous()):
            c = _blank(fa, 2, 16, 3, 64)
            q = fa.cache_append(c, t, t, torch.tensor([[1, 0]]).int().cuda(), torch.arange(9).int().cuda() + 11,
                                torch.zeros(9).int().cuda(), Q=t, table=table, interleaved=inter)
            got.append((q, *_cpu(c)))
        for a, b in zip(*got):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert fa.status_query() == fa.OK


@pytest.mark.parametrize("case", APPEND)
def test_append_and_gather(fa, cuda, case):
    page, hk, hq, D, r, dtype, inter, ocp = case
    counts, starts = [1, 0, 37, 150], [0, 5, 63, 20]
    per_seq = -(-max(a + b for a, b in zip(counts, starts)) // page)
    cache = _blank(fa, 4 * per_seq + 2, page, hk, D)
    bt = _tables(3, 4, per_seq, 4 * per_seq + 2)
    n = sum(counts)
    qkv = torch.randn(n, hq + 2 * hk, D, generator=_gen(9)).to(dtype)
    qkv[0] = 0.0
    seq = torch.repeat_interleave(torch.arange(4), torch.tensor(counts)).int()
    pos = torch.cat([torch.arange(s, s + c) for s, c in zip(starts, counts)]).int()
    order = torch.randperm(n, generator=_gen(10))  # tokens in any order
    qkv, seq, pos = qkv[order], seq[order], pos[order]
    d = qkv.cuda()
    table = fa.rotary_table(300, r) if r else None
    before = _cpu(cache)
    q = fa.cache_append(cache, d[:, hq:hq + hk], d[:, hq + hk:], bt.cuda(), pos.cuda(), seq.cuda(), Q=d[:, :hq],
                        table=table, interleaved=inter, scale_mode="ocp" if ocp else "reference")
    assert fa.status_query() == fa.OK

    def turned(x):  # [n, heads, D] as [1, heads, n, D]
        if not r:
            return x.contiguous()
        return fa.rotary(x.transpose(0, 1)[None], table, pos.cuda(), interleaved=inter)[0].transpose(0, 1).contiguous()

    assert torch.equal(q, turned(d[:, :hq]))
    # Keys: the oracle's codes of the separately rotated keys, byte for byte.
    codes, scales = oracle.quantize(turned(d[:, hq:hq + hk]).cpu().float().numpy(), int(ocp))
    codes, scales = torch.from_numpy(oracle.pack_codes(codes)), torch.from_numpy(scales)
    at, off = bt.long()[seq.long(), pos.long() // page], pos.long() % page
    want = [t.clone() for t in before]
    want[0][at, :, off], want[1][at, :, off], want[2][at, :, off] = codes, scales, qkv[:, hq + hk:].half()
    got = _cpu(cache)
    for g, w in zip(got, want):  # and nothing else of the cache is touched
        assert torch.equal(g.view(torch.uint8), w.view(torch.uint8))
    # Read back, each head twice, in both types.
    for out in (F16, F32):
        K, V = fa.cache_gather(cache, bt.cuda(), torch.tensor(starts).int().cuda(), torch.tensor(counts).int().cuda(),
                               max(counts), heads=2 * hk, dtype=out)
        for s in range(4):
            k, v = ref.read(got, bt[s], starts[s], counts[s])
            for h in range(2 * hk):
                assert torch.equal(K[s, h, :counts[s]].cpu(), k[h // 2].to(out))
                assert torch.equal(V[s, h, :counts[s]].cpu(), v[h // 2].to(out))
            assert not K[s, :, counts[s]:].any() and not V[s, :, counts[s]:].any()
    assert fa.status_query() == fa.OK


def test_append_special_values(fa, cuda):
    """Infinities, NaN, -0.0, subnormals and exact ties enter the cache as the quantiser has them (255 as 254)."""
    for dtype in (F16, F32):
        x = torch.randn(4, 1, 64, generator=_gen(2)).to(dtype)
        x[0, 0, :8] = torch.tensor([math.inf, -math.inf, math.nan, -0.0, 0.25, 2.5, -5.0, 1.25])
        x[1, 0, :32] = 0.0
        x[1, 0, 32:] = 2.0 ** -24
        x[2, 0, :32] = torch.tensor([0.25, -0.25, 0.75, 1.0] * 8)
        if dtype == F32:
            x[3, 0, 3] = 3e38   # 2^128: the scale byte is 255
        cache = _blank(fa, 1, 16, 1, 64)
        fa.cache_append(cache, x.cuda(), x.cuda(), torch.zeros(1, 1).int().cuda(), torch.arange(4).int().cuda(),
                        torch.zeros(4).int().cuda())
        codes, scales = fa.quantize(x.cuda())
        assert torch.equal(cache.k_codes[0, 0, :4], codes[:, 0])
        assert torch.equal(cache.k_scales[0, 0, :4], scales[:, 0].clamp(max=254))
        got, want = cache.v[0, 0, :4].cpu(), x[:, 0].half()
        same = got.view(torch.int16) == want.view(torch.int16)
        if dtype == F32:  # (converting leaves a NaN's payload open)
            same |= got.isnan() & want.isnan()
        assert bool(same.all())
        assert fa.status_query() == fa.OK


def test_append_padding_and_bad_indices(fa, cuda):
    cache = _blank(fa, 4, 16, 2, 64)
    before = _cpu(cache)
    x = torch.randn(3, 2, 64, generator=_gen(2)).half().cuda()
    bt = torch.tensor([[1, 2], [3, 0], [9, -1]], dtype=torch.int32).cuda()
    table = fa.rotary_table(40, 64)

    def put(pos, ids=None, t=None):
        pos = torch.tensor(pos, dtype=torch.int32).cuda()
        ids = None if ids is None else torch.tensor(ids, dtype=torch.int32).cuda()
        return fa.cache_append(cache, x, x, bt, pos, ids, Q=x, table=t)

    q = put([-1, -1, -7])                               # padding only
    assert not q.any() and fa.status_query() == fa.OK
    for pos, ids, t, word in (([-1, -1, 3], None, None, b"page 9"), ([-1, -1, 20], None, None, b"page -1"),
                              ([32, -1, -1], None, None, b"length"), ([-1, 0, -1], [0, 3, 0], None, b"sequence 3"),
                              ([-1, 0, -1], [0, -2, 0], None, b"sequence -2")):
        put(pos, ids, t)
        assert fa.status_query() == fa.EINDEX
        assert word in fa.lib().fp4attn_last_error(), word
    short = fa.rotary_table(4, 64)
    q = put([4, -1, -1], None, short)
    assert fa.status_query() == fa.EINDEX and b"position 4" in fa.lib().fp4attn_last_error()
    assert not q.any()
    for g, w in zip(_cpu(cache), before):
        assert torch.equal(g.view(torch.uint8), w.view(torch.uint8))
    put([-1, 17, -1], None, table)                      # the good token of a batch is written
    assert fa.status_query() == fa.OK
    assert torch.equal(cache.v[0, :, 1], x[1])


def test_gather_bad_indices(fa, cuda):
    cache = _blank(fa, 4, 16, 1, 32, fill=False)
    i = lambda *v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    bt = torch.tensor([[0, 4]], dtype=torch.int32).cuda()
    for start, length in ((-1, 3), (0, 9), (0, -2), (30, 8), (10, 8), (2147483640, 8)):
        K, V = fa.cache_gather(cache, bt, i(start), i(length), 8)
        assert fa.status_query() == fa.EINDEX, (start, length)
    assert fa.cache_gather(cache, bt, None, i(0), 0)[0].shape == (1, 1, 0, 32)
    assert fa.status_query() == fa.OK


# ------------------------------------------------------------------------------- attention
def _filled(fa, seed, pages, page, hk, D, ocp=False):
    """A cache of random codes, scales around 2 and normal values, every place used."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = fa.PagedCache.empty(pages, page, hk, D)
    c.k_codes.copy_(torch.randint(0, 256, c.k_codes.shape, generator=g, device="cuda"))
    c.k_scales.copy_(torch.randint(125, 128, c.k_scales.shape, generator=g, device="cuda"))
    c.v.normal_(generator=g)
    return c


def _poison_behind(c, bt, lens):
    """NaN and infinite scales and values in every place no sequence uses."""
    P, H, page, D = c.v.shape
    used = torch.zeros(P, page, dtype=torch.bool)
    for row, n in zip(bt.tolist(), lens):
        for p in range(n):
            used[row[p // page], p % page] = True
    free = (~used).cuda()[:, None, :].expand(P, H, page)
    c.k_scales[free] = 255
    c.v[free] = math.nan


def _check_attention(fa, c, q, bt, lens, ocp, out_dtype, scale=None, poison=True, **kw):
    if poison:
        _poison_behind(c, bt, lens)
    out, lse = fa.paged_attention_lse(q.cuda(), c, bt.cuda(), torch.tensor(lens).int().cuda(), softmax_scale=scale,
                                      scale_mode="ocp" if ocp else "reference", out_dtype=out_dtype, **kw)
    assert fa.status_query() == fa.OK
    assert out.dtype == out_dtype and out.is_contiguous()
    qq, host = ref.quantized(q.contiguous(), ocp), _cpu(c)
    for b, n in enumerate(lens):
        k, v = ref.read(host, bt[b], 0, n)
        want, want_lse, size = ref.attend(qq[b], k, v, scale)
        got, got_lse = out[b].cpu().double(), lse[b].cpu().double()
        if n == 0:
            assert not got.any() and bool((got_lse == math.inf).all())
            continue
        g = q.shape[1] // k.shape[0]
        z = torch.einsum("hgd,hnd->hgn", qq[b].view(k.shape[0], g, -1), k) * (scale or 1 / math.sqrt(q.shape[2]))
        zmax = float(z.abs().max())
        off = (got - want).abs()
        bound = ref.attend_bound(want, size, n, float(v.abs().max()), zmax, out_dtype)
        assert bool((off <= bound).all()), (b, n, float((off / bound).max()))
        assert bool(((got_lse - want_lse).abs() <= ref.lse_bound(want_lse, n, zmax)).all()), (b, n)
    return out, lse


ATTEND = [  # page, kv_heads, group, D
    (64, 2, 4, 128),
    (16, 1, 1, 64),
    (32, 3, 7, 96),
    (128, 2, 16, 128),
    (16, 2, 5, 32),
    (64, 1, 3, 160),
    (32, 2, 8, 256),
    (64, 1, 40, 128),
    (16, 1, 17, 64),
]


@pytest.mark.parametrize("out_dtype,in_dtype,ocp", [(F16, F16, False), (F32, F16, True), (F32, F32, False)])
@pytest.mark.parametrize("shape", ATTEND)
def test_attention(fa, cuda, shape, out_dtype, in_dtype, ocp):
    """Lengths around every border of pages and of 128-key tiles, and none at all."""
    page, hk, g, D = shape
    lens = [1, 0, 15, 16, 17, 64, 127, 128, 129, 255, 256, 300, 777]
    per_seq = -(-max(lens) // page) + 1
    pages = len(lens) * per_seq + 1
    c = _filled(fa, 1, pages, page, hk, D)
    q = torch.randn(len(lens), hk * g, D, generator=_gen(2)).to(in_dtype)
    _check_attention(fa, c, q, _tables(3, len(lens), per_seq, pages), lens, ocp, out_dtype)


@pytest.mark.parametrize("out_dtype", [F16, F32])
@pytest.mark.parametrize("batch,hk,g,n", [(1, 1, 8, 30001), (1, 8, 4, 5000), (3, 2, 4, 9000), (1, 1, 1, 20000)])
def test_attention_over_long_sequences(fa, cuda, batch, hk, g, n, out_dtype):
    """Sequences whose keys are split over many SMs and joined."""
    lens = [n - 1111 * i for i in range(batch)]
    per_seq = -(-n // 64)
    c = _filled(fa, 5, batch * per_seq, 64, hk, 128)
    q = torch.randn(batch, hk * g, 128, generator=_gen(6)).half()
    _check_attention(fa, c, q, _tables(7, batch, per_seq, batch * per_seq), lens, False, out_dtype)


def test_attention_over_many_sequences(fa, cuda):
    """More (sequence, head) pairs than SMs, of unequal length, some empty."""
    g = _gen(3)
    lens = [int(x) for x in torch.randint(0, 400, (90,), generator=g)]
    lens[4] = lens[5] = lens[6] = 0
    per_seq, hk = 25, 3
    c = _filled(fa, 5, 90 * per_seq, 16, hk, 64)
    q = torch.randn(90, hk * 2, 64, generator=g).half()
    bt = _tables(7, 90, per_seq, 90 * per_seq)
    _check_attention(fa, c, q, bt, lens, False, F16)
    # all empty
    zero = torch.zeros(90).int().cuda()
    out, lse = fa.paged_attention_lse(q.cuda(), c, bt.cuda(), zero)
    assert not out.any() and bool((lse == math.inf).all()) and fa.status_query() == fa.OK


@pytest.mark.parametrize("out_dtype", [F16, F32])
@pytest.mark.parametrize("order", ["rising", "falling", "spike"])
def test_attention_when_the_maximum_moves(fa, cuda, order, out_dtype):
    """Scores that grow by far more than FP16's range along the sequence, fall, or have one key above all."""
    n, D = 1500, 64
    c = _filled(fa, 5, 24, 64, 1, D)
    q = torch.randn(1, 4, D, generator=_gen(6)).half()
    bt = torch.arange(24).int()[None]
    for p in range(24):  # page p's keys: scale 2^(p/3 - 4), or one key of 2^6
        e = {"rising": 123 + p // 3, "falling": 131 - p // 3, "spike": 121}[order]
        c.k_scales[p] = e
    if order == "spike":
        c.k_scales[11, :, 17] = 133
    _check_attention(fa, c, q, bt, [n], False, out_dtype)


@pytest.mark.parametrize("scale", [1.0, 0.01, 3.0])
def test_attention_softmax_scale(fa, cuda, scale):
    c = _filled(fa, 5, 10, 64, 2, 64)
    q = torch.randn(2, 4, 64, generator=_gen(6)).half()
    _check_attention(fa, c, q, _tables(1, 2, 5, 10), [300, 77], False, F32, scale=scale)


def test_attention_extreme_scales(fa, cuda):
    """Key scales from 2^-127 on, and equal scores everywhere: the plain mean."""
    c = _filled(fa, 5, 5, 64, 1, 64)
    c.k_scales.fill_(0)
    q = torch.randn(1, 2, 64, generator=_gen(6)).half()
    _check_attention(fa, c, q, torch.arange(5).int()[None], [317], False, F32)


def test_attention_strides(fa, cuda):
    """A query inside a fused projection, pages inside a larger tensor, rows of a wider block table."""
    D, hk, page = 128, 2, 32
    big_v = torch.randn(20, 3, hk, page, D, generator=_gen(1)).half().cuda()
    big_c = torch.randint(0, 256, (20, 3, hk, page, D // 2), generator=_gen(2)).to(torch.uint8).cuda()
    big_s = torch.randint(125, 128, (20, 3, hk, page, D // 32), generator=_gen(3)).to(torch.uint8).cuda()
    c = fa.PagedCache(big_c[:, 1], big_s[:, 1], big_v[:, 1])
    qkv = torch.randn(2, 8 + 2 * hk, D, generator=_gen(4)).half()
    bt = _tables(5, 2, 10, 20)
    wide = torch.full((2, 16), 7, dtype=torch.int32)
    wide[:, :10] = bt
    lens = torch.tensor([300, 111]).int().cuda()
    want = fa.paged_attention(qkv[:, :8].contiguous().cuda(), fa.PagedCache(*(t[:, 1].contiguous() for t in (big_c, big_s, big_v))),
                              bt.cuda(), lens)
    got = fa.paged_attention(qkv.cuda()[:, :8], c, wide.cuda()[:, :10], lens)
    assert torch.equal(got, want)
    _check_attention(fa, c, qkv[:, :8], bt, [300, 111], False, F16, poison=False)


def test_attention_is_the_forward_of_one_row(fa, cuda):
    """What fused_fp4_attention gives for one query over the same tokens."""
    B, H, D, n = 2, 4, 128, 200
    K, V = (torch.randn(B, H, n, D, generator=_gen(i)).half().cuda() for i in (1, 2))
    Q = torch.randn(B, H, 1, D, generator=_gen(3)).half().cuda()
    c = _blank(fa, 8, 64, H, D)
    bt = torch.arange(8).int().view(2, 4).cuda()
    ids = torch.repeat_interleave(torch.arange(2), n).int().cuda()
    pos = torch.arange(n).int().repeat(2).cuda()
    fa.cache_append(c, K.transpose(1, 2).reshape(B * n, H, D), V.transpose(1, 2).reshape(B * n, H, D), bt, pos, ids)
    out, lse = fa.paged_attention_lse(Q[:, :, 0], c, bt, torch.full((2,), n).int().cuda(), out_dtype=F32)
    want, want_lse = fa.fused_fp4_attention_lse(Q, K, V, out_dtype=F32)
    # (the forward rounds P to FP16 and sums the rounded values)
    assert float((out - want[:, :, 0]).abs().max()) <= 2e-3
    assert float((lse - want_lse[:, :, 0]).abs().max()) <= 2e-3
    k, v = fa.cache_gather(c, bt, None, torch.full((2,), n).int().cuda(), n)
    assert torch.equal(v, V)
    assert torch.equal(fa.debug_scores(Q, k), fa.debug_scores(Q, K))  # quantising the read keys again changes nothing


def test_attention_bad_indices(fa, cuda):
    c = _filled(fa, 5, 4, 64, 1, 64)
    q = torch.randn(2, 2, 64, generator=_gen(6)).half().cuda()
    good = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32).cuda()
    lens = torch.tensor([100, 128], dtype=torch.int32).cuda()
    want = fa.paged_attention(q, c, good, lens)
    for bt, ln in (([[0, 4], [2, 3]], [100, 128]), ([[0, -1], [2, 3]], [100, 128]), ([[0, 1], [2, 3]], [129, 128]),
                   ([[0, 1], [2, 3]], [-5, 128])):
        got = fa.paged_attention(q, c, torch.tensor(bt, dtype=torch.int32).cuda(), torch.tensor(ln, dtype=torch.int32).cuda())
        assert fa.status_query() == fa.EINDEX
        assert torch.equal(got[1], want[1])           # the other sequence has its result
    assert torch.equal(fa.paged_attention(q, c, good, lens), want) and fa.status_query() == fa.OK


def test_attention_repeats_bit_for_bit(fa, cuda):
    lens = torch.tensor([4000, 3, 0, 1234]).int().cuda()
    c = _filled(fa, 5, 260, 64, 2, 128)
    bt = _tables(1, 4, 65, 260).cuda()
    q = torch.randn(4, 8, 128, generator=_gen(6)).half().cuda()
    ws = torch.empty(fa.paged_attention_workspace_size(c, 4, 8), dtype=torch.uint8, device="cuda")
    out = torch.empty_like(q)
    first, lse = fa.paged_attention_lse(q, c, bt, lens)
    for fill in (0, 255, 1):
        ws.fill_(fill)                                # any content
        got, l2 = fa.paged_attention_lse(q, c, bt, lens, out=out, workspace=ws)
        assert got is out and torch.equal(out, first) and torch.equal(lse, l2)
    assert fa.status_query() == fa.OK


def test_attention_writes_nothing_else(fa, cuda):
    c = _filled(fa, 5, 40, 64, 2, 128)
    bt = _tables(1, 3, 13, 40).cuda()
    q = torch.randn(3, 8, 128, generator=_gen(6)).half().cuda()
    size = fa.paged_attention_workspace_size(c, 3, 8)
    ws = torch.full((size + 512,), 0xA5, dtype=torch.uint8, device="cuda")
    buf = torch.full((3 * 8 * 128 + 256,), 7.0, dtype=F16, device="cuda")
    fa.paged_attention(q, c, bt, torch.tensor([800, 0, 5]).int().cuda(), out=buf[128:-128].view(3, 8, 128),
                       workspace=ws[256:256 + size])
    assert fa.status_query() == fa.OK
    assert bool((ws[:256] == 0xA5).all()) and bool((ws[256 + size:] == 0xA5).all())
    assert bool((buf[:128] == 7).all()) and bool((buf[-128:] == 7).all())


def test_attention_captured_with_growing_lengths(fa, cuda):
    """A decode step captured once: append and attend, replayed while the lengths grow in place."""
    D, hk, g, B = 64, 2, 4, 3
    c = _blank(fa, 30, 16, hk, D)
    bt = _tables(2, B, 10, 30).cuda()
    kv = torch.randn(40, B, 2 * hk, D, generator=_gen(1)).half().cuda()
    qs = torch.randn(40, B, hk * g, D, generator=_gen(2)).half().cuda()
    table = fa.rotary_table(256, D)
    q, k, v = qs[0].clone(), kv[0, :, :hk].clone(), kv[0, :, hk:].clone()
    pos, lens = torch.zeros(B).int().cuda(), torch.ones(B).int().cuda()
    ws = torch.empty(fa.paged_attention_workspace_size(c, B, hk * g), dtype=torch.uint8, device="cuda")

    def step():
        turned = fa.cache_append(c, k, v, bt, pos, Q=q, table=table)
        return fa.paged_attention(turned, c, bt, lens, workspace=ws)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for t in range(40):
        q.copy_(qs[t]), k.copy_(kv[t, :, :hk]), v.copy_(kv[t, :, hk:])
        pos.fill_(t), lens.fill_(t + 1)
        graph.replay()
        assert torch.equal(out, fa.paged_attention(fa.rotary(q.transpose(0, 1)[None], table, pos)[0].transpose(0, 1).contiguous(),
                                                   c, bt, lens))
    assert fa.status_query() == fa.OK


def test_two_captured_calls_share_a_workspace(fa, cuda):
    """Graphs of different calls over one workspace, replayed in turn: each gives its own result every time."""
    c = _filled(fa, 5, 400, 64, 2, 128)
    bt = _tables(1, 4, 100, 400).cuda()
    ws = torch.empty(fa.paged_attention_workspace_size(c, 4, 8), dtype=torch.uint8, device="cuda")
    calls = []
    for seed, lens in ((1, [6000, 3, 0, 1234]), (2, [1, 6400, 6400, 77])):
        q, ln = torch.randn(4, 8, 128, generator=_gen(seed)).half().cuda(), torch.tensor(lens).int().cuda()
        want = fa.paged_attention(q, c, bt, ln)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = fa.paged_attention(q, c, bt, ln, workspace=ws)
        calls.append((graph, out, want, q, ln))  # (the graph reads q and ln where they are)
    for _ in range(3):
        for graph, out, want, *_ in calls:
            out.zero_()
            graph.replay()
            assert torch.equal(out, want)
    assert fa.status_query() == fa.OK


def test_caches_past_32_bit_offsets(fa, cuda):
    """Pages whose values, codes and scales lie 4 GiB and more into their tensors."""
    P, hk, page, D = 70000, 8, 64, 128              # 9.2 GB of values, 2.3 GB of codes
    c = fa.PagedCache.empty(P, page, hk, D)
    bt = torch.tensor([[P - 1, 5, P - 3], [P - 2, 40000, 33000]], dtype=torch.int32)
    n = 3 * page - 7
    kv = torch.randn(2 * n, 2 * hk, D, generator=_gen(1)).half()
    pos, ids = torch.arange(n).int().repeat(2), torch.repeat_interleave(torch.arange(2), n).int()
    d = kv.cuda()
    fa.cache_append(c, d[:, :hk], d[:, hk:], bt.cuda(), pos.cuda(), ids.cuda())
    lens = torch.full((2,), n).int().cuda()
    K, V = fa.cache_gather(c, bt.cuda(), None, lens, n)
    assert torch.equal(V, d[:, hk:].view(2, n, hk, D).transpose(1, 2))
    q = torch.randn(2, hk, D, generator=_gen(2)).half()
    out = fa.paged_attention(q.cuda(), c, bt.cuda(), lens, out_dtype=F32)
    fa.copy_pages([c], [P - 1, P - 2], [P - 4, 1])
    moved = torch.tensor([[P - 4, 5, P - 3], [1, 40000, 33000]], dtype=torch.int32)
    assert torch.equal(out, fa.paged_attention(q.cuda(), c, moved.cuda(), lens, out_dtype=F32))
    small = fa.PagedCache(*(t[bt.flatten().long().cuda()].contiguous() for t in (c.k_codes, c.k_scales, c.v)))
    assert torch.equal(out, fa.paged_attention(q.cuda(), small, torch.arange(6).int().view(2, 3).cuda(), lens, out_dtype=F32))
    assert fa.status_query() == fa.OK


def test_attention_on_two_streams(fa, cuda):
    """Calls in flight on two streams at once, outputs and workspaces their own."""
    c = _filled(fa, 5, 200, 64, 2, 128)
    bt = _tables(1, 4, 50, 200).cuda()
    lens = torch.tensor([3000, 100, 1, 2222]).int().cuda()
    qs = [torch.randn(4, 8, 128, generator=_gen(i)).half().cuda() for i in range(8)]
    want = [fa.paged_attention(q, c, bt, lens) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [fa.paged_attention(q, c, bt, lens, stream=streams[i % 2]) for i, q in enumerate(qs)]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert fa.status_query() == fa.OK


def test_attention_writes_over_its_queries(fa, cuda):
    """out=Q gives the plain call's bytes; an output half over Q is refused."""
    cache = fa.PagedCache.empty(40, 16, 2, 64)
    table = torch.arange(40, device="cuda", dtype=torch.int32).view(2, 20)
    lens = torch.tensor([300, 17], device="cuda", dtype=torch.int32)
    seq = torch.arange(2, device="cuda", dtype=torch.int32).repeat_interleave(320)
    K, V = (torch.randn(640, 2, 64, generator=_gen(s)).half().cuda() for s in (8, 9))
    fa.cache_append(cache, K, V, table, torch.arange(320, device="cuda", dtype=torch.int32).repeat(2), seq_ids=seq)
    base = torch.randn(3, 4, 64, generator=_gen(10)).half().cuda()
    want = fa.paged_attention(base[:2].clone(), cache, table, lens)
    with pytest.raises(ValueError, match="partly"):
        fa.paged_attention(base[:2], cache, table, lens, out=base[1:])
    fa.paged_attention(base[:2], cache, table, lens, out=base[:2])
    assert torch.equal(base[:2], want)


def test_attention_refuses_mismatched_tensors(fa, cuda):
    c = _filled(fa, 5, 4, 64, 2, 64)
    q = torch.randn(2, 4, 64).half().cuda()
    bt, lens = torch.zeros(2, 2).int().cuda(), torch.ones(2).int().cuda()
    for bad in (dict(Q=q[:, :3]), dict(Q=q.bfloat16()), dict(Q=q[..., :32]), dict(block_table=bt[:1]),
                dict(block_table=bt.long()), dict(seq_lens=lens.cpu()), dict(seq_lens=lens[:1]),
                dict(scale_mode="other"), dict(out=torch.empty(2, 4, 64)), dict(workspace=torch.empty(8).cuda()),
                dict(workspace=torch.empty(0, dtype=torch.uint8).cuda())):
        args = dict(Q=q, cache=c, block_table=bt, seq_lens=lens)
        args.update(bad)
        with pytest.raises((ValueError, TypeError, fa.Fp4AttnError)):
            fa.paged_attention(**args)
    with pytest.raises(ValueError):
        fa.PagedCache(c.k_codes, c.k_scales, c.v[:, :1])
    with pytest.raises(ValueError):
        fa.PagedCache(c.k_codes, c.k_scales, c.v.transpose(1, 2))
    assert fa.paged_attention(q[:0], c, bt[:0], lens[:0]).shape == (0, 4, 64)
    assert fa.status_query() == fa.OK


# ------------------------------------------------------------------------------- page copies
@pytest.mark.parametrize("layers,n,page,hk,D", [(1, 1, 64, 2, 128), (3, 5, 16, 1, 32), (9, 70, 16, 3, 96), (2, 300, 32, 1, 160)])
def test_copy_pages(fa, cuda, layers, n, page, hk, D):
    pages = 2 * n + 3
    caches = [_filled(fa, i, pages, page, hk, D) for i in range(layers)]
    want = [_cpu(c) for c in caches]
    order = torch.randperm(pages, generator=_gen(1))
    src, dst = order[:n].clone(), order[n:2 * n]
    src[n // 2:] = src[0]                              # one page to several
    for w in want:
        for t in w:
            t[dst] = t[src]
    fa.copy_pages(caches, src, dst)
    assert fa.status_query() == fa.OK
    for c, w in zip(caches, want):
        for g, t in zip(_cpu(c), w):
            assert torch.equal(g.view(torch.uint8), t.view(torch.uint8))


def test_copy_pages_refuses(fa, cuda):
    c = _filled(fa, 1, 4, 16, 1, 32)
    for src, dst in (([0], [4]), ([0, 1], [2, 2]), ([0], [0]), ([0, 1], [1, 2]), ([0], [2 ** 32])):
        with pytest.raises((fa.Fp4AttnError, ValueError)):
            fa.copy_pages([c], src, dst)
    with pytest.raises(ValueError):
        fa.copy_pages([c], torch.tensor([0]).cuda(), [1])
    with pytest.raises(ValueError):
        fa.copy_pages([c], [0, 1], [2])
    fa.copy_pages([c], [], [])


def test_copy_pages_with_gaps_between_pages(fa, cuda):
    big = torch.randn(6, 2, 1, 16, 32, generator=_gen(1)).half().cuda()
    c = _filled(fa, 1, 6, 16, 1, 32)
    view = fa.PagedCache(c.k_codes, c.k_scales, big[:, 1])
    want = big.clone()
    want[5, 1] = want[0, 1]
    fa.copy_pages([view], [0], [5])
    assert torch.equal(big, want) and fa.status_query() == fa.OK


# ------------------------------------------------------------------------------- all together
@pytest.mark.parametrize("dim,rot,page,interleaved", [(128, 128, 64, False), (96, 32, 16, True)])
def test_serving_run(fa, cuda, dim, rot, page, interleaved):
    """Two prompts attended and appended, one forked, twelve tokens decoded by
    every sequence with copies on write, one freed, the cache compacted, and
    eight more tokens: every decoded output against the 64-bit attention over
    that sequence's own keys and values."""
    layers, hq, hk = 2, 4, 2
    pool = fa.PagePool(64, page)
    caches = [_blank(fa, 64, page, hk, dim) for _ in range(layers)]
    table = fa.rotary_table(512, rot, scaling="yarn", factor=2.0, original_positions=256)
    g = _gen(11)
    truth = {}  # sequence -> per layer ([keys], [values]) of [hk, dim] float64

    def tokens(n):
        return torch.randn(n, hq + 2 * hk, dim, generator=g).half()

    def remember(seq, layer, x, first):
        pos = torch.arange(first, first + x.shape[0])
        k = fa.rotary(x[:, hq:hq + hk].cuda().transpose(0, 1)[None], table, pos.int().cuda(), interleaved)[0].transpose(0, 1)
        truth[seq][layer][0].extend(ref.quantized(k.cpu().contiguous()))
        truth[seq][layer][1].extend(x[:, hq + hk:].double())

    seqs = []
    for n in (page + 5, 3):
        seq = pool.new()
        seqs.append(seq)
        truth[seq] = [([], []) for _ in range(layers)]
        fa.copy_pages(caches, *pool.extend(seq, n))
        bt = pool.block_table([seq], "cuda")
        pos, ids = torch.arange(n).int().cuda(), torch.zeros(n).int().cuda()
        for layer, c in enumerate(caches):
            x = tokens(n)
            d = x.cuda()
            q = fa.cache_append(c, d[:, hq:hq + hk], d[:, hq + hk:], bt, pos, ids, Q=d[:, :hq], table=table,
                                interleaved=interleaved)
            remember(seq, layer, x, 0)
            # the prompt's own attention, over the keys as the cache has them
            K, V = fa.cache_gather(c, bt, None, torch.tensor([n]).int().cuda(), n, heads=hq)
            out = fa.fused_fp4_attention(q.transpose(0, 1)[None].contiguous(), K, V, causal=True, out_dtype=F32)[0]
            kk, vv = (torch.stack(t, 1) for t in truth[seq][layer])
            qq = ref.quantized(q.cpu())
            for i in range(n):
                want, _, _ = ref.attend(qq[i], kk[:, :i + 1], vv[:, :i + 1])
                assert float((out[:, i].cpu().double() - want).abs().max()) <= 2e-2  # the forward's tolerance

    def decode():
        first = [pool.length(s) for s in seqs]
        for s in seqs:
            fa.copy_pages(caches, *pool.extend(s, 1))
        bt = pool.block_table(seqs, "cuda")
        pos = torch.tensor(first).int().cuda()
        for layer, c in enumerate(caches):
            x = tokens(len(seqs))
            d = x.cuda()
            q = fa.cache_append(c, d[:, hq:hq + hk], d[:, hq + hk:], bt, pos, Q=d[:, :hq], table=table,
                                interleaved=interleaved)
            out = fa.paged_attention(q, c, bt, pos + 1)
            qq = ref.quantized(q.cpu())
            for i, s in enumerate(seqs):
                remember(s, layer, x[i:i + 1], first[i])
                k, v = (torch.stack(t, 1) for t in truth[s][layer])
                want, _, size = ref.attend(qq[i], k, v)
                z = torch.einsum("hgd,hnd->hgn", qq[i].view(hk, hq // hk, dim), k) / math.sqrt(dim)
                bound = ref.attend_bound(want, size, k.shape[1], float(v.abs().max()), float(z.abs().max()), F16)
                assert bool(((out[i].cpu().double() - want).abs() <= bound).all())

    child = pool.fork(seqs[0])
    truth[child] = [(list(k), list(v)) for k, v in truth[seqs[0]]]
    seqs.append(child)
    for _ in range(12):
        decode()
    pool.free(seqs[0])
    seqs = seqs[1:]
    src, dst = pool.compact()
    fa.copy_pages(caches, src, dst)
    for _ in range(8):
        decode()
    assert fa.status_query() == fa.OK
