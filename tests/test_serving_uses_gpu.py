"""Uses of the serving calls that the rest of the tests do not make: the gradient in the
training type, prompt chunks behind a cached prefix, several new tokens of one sequence as
rows that share its pages, and more sequences than a scan of the lengths takes at once."""
import math

import pytest
import torch

import serving_ref as ref

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32


def _gen(seed):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------------------------- rotary, FP16
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rot", [(128, 128), (64, 30), (96, 48), (128, 50)])
def test_rotary_gradient_in_fp16(fa, cuda, dim, rot, interleaved):
    B, H, S = 2, 3, 21
    table = fa.rotary_table(300, rot, scaling="yarn", factor=4.0, original_positions=128)
    pos = torch.randint(0, 300, (B, S), generator=_gen(7)).int()
    x = torch.randn(B, S, H, dim, generator=_gen(5)).half().cuda().transpose(1, 2).requires_grad_()
    dy = torch.randn(B, H, S, dim, generator=_gen(6)).half()
    y = fa.rotary_embedding(x, table, pos.cuda(), interleaved=interleaved)
    (dx,) = torch.autograd.grad(y, x, dy.cuda())
    assert y.dtype == dx.dtype == F16
    cos, sin = ref.angles(table.cpu(), pos[:, None])
    for got, of, s in ((y, x.detach().cpu(), sin), (dx, dy, -sin)):
        want, size = ref.rotate(of, cos, s, interleaved)
        assert bool(((got.detach().cpu().double() - want).abs() <= ref.rotary_bound(want, size, F16)).all())
    # the same by the plain call that turns back
    assert torch.equal(dx, fa.rotary(dy.cuda(), table, pos.cuda(), interleaved, inverse=True))
    # Differences: <dy, R(x + v) - R(x - v)> / 2 = <dx, v>.  x, v in steps of 2^-6 below 8, so that x + v
    # and x - v are exact; then each y and dx is off by its bound, weighted by dy or v.
    grid = (torch.randn(2, B, H, S, dim, generator=_gen(8)).clamp(-3, 3) * 64).round() / 64
    a, v = grid[0].half(), grid[1].half()
    ends, slack = [], 0.0
    for t in (a + v, a - v):
        ends.append(fa.rotary(t.cuda(), table, pos.cuda(), interleaved).cpu().double())
        want, size = ref.rotate(t, cos, sin, interleaved)
        slack += float((ref.rotary_bound(want, size, F16) * dy.double().abs()).sum()) / 2
    want, size = ref.rotate(dy, cos, -sin, interleaved)
    slack += float((ref.rotary_bound(want, size, F16) * v.double().abs()).sum())
    got = float((dx.cpu().double() * v.double()).sum())
    assert abs(float(((ends[0] - ends[1]) / 2 * dy.double()).sum()) - got) <= slack * (1 + 1e-9)


# ------------------------------------------------------------------------------- chunks
def _prompt(fa, n, hk, hq, dim, page, seed, rot):
    """A prompt of n tokens in the cache, in chunks: (cache, block table, rotated queries, raw rows)."""
    pages = -(-n // page) + 3
    cache = fa.PagedCache.empty(pages, page, hk, dim)
    cache.k_scales.fill_(255), cache.v.fill_(math.nan)
    bt = torch.randperm(pages, generator=_gen(seed))[: -(-n // page)].int()[None].cuda()
    rows = torch.randn(n, hq + 2 * hk, dim, generator=_gen(seed + 1)).half().cuda()
    table = fa.rotary_table(n, rot)
    q = []
    for first in range(0, n, 37):
        x = rows[first:first + 37]
        at = torch.arange(first, first + len(x), dtype=torch.int32, device="cuda")
        q.append(fa.cache_append(cache, x[:, hq:hq + hk], x[:, hq + hk:], bt, at, seq_ids=torch.zeros_like(at), Q=x[:, :hq],
                                 table=table))
    return cache, bt, torch.cat(q), table


def _truth(cache, bt, n):
    return ref.read((cache.k_codes.cpu(), cache.k_scales.cpu(), cache.v.cpu()), bt[0].cpu(), 0, n)


@pytest.mark.parametrize("hk,hq,dim,page,prefix,chunk", [(2, 4, 128, 64, 150, 70), (1, 8, 64, 16, 33, 40),
                                                        (3, 3, 96, 32, 1, 131), (2, 4, 64, 128, 128, 1)])
def test_a_chunk_behind_a_cached_prefix(fa, cuda, hk, hq, dim, page, prefix, chunk):
    """A prompt chunk by way of cache_gather and the causal forward (its queries are the last of the keys): every
    row against the 64-bit attention over the tokens before it, at the forward's tolerance."""
    n = prefix + chunk
    cache, bt, q, _ = _prompt(fa, n, hk, hq, dim, page, 11, dim)
    length = torch.tensor([n], dtype=torch.int32, device="cuda")
    K, V = fa.cache_gather(cache, bt, None, length, n, heads=hq)
    out = fa.fused_fp4_attention(q[prefix:].transpose(0, 1)[None].contiguous(), K, V, causal=True, out_dtype=F32)[0]
    k, v = _truth(cache, bt, n)
    qq = ref.quantized(q[prefix:].cpu())
    for i in range(chunk):
        want, _, _ = ref.attend(qq[i], k[:, :prefix + i + 1], v[:, :prefix + i + 1])
        assert float((out[:, i].cpu().double() - want).abs().max()) <= 2e-2
    assert fa.status_query() == fa.OK


@pytest.mark.parametrize("out_dtype", [F16, F32])
@pytest.mark.parametrize("hk,hq,dim,page,n,new", [(2, 4, 128, 64, 200, 5), (1, 8, 64, 16, 130, 131), (2, 6, 96, 32, 500, 300)])
def test_new_tokens_of_one_sequence_as_rows(fa, cuda, hk, hq, dim, page, n, new, out_dtype):
    """The last `new` tokens of a sequence as rows that share its pages, with lengths that grow by one."""
    new = min(new, n)
    cache, bt, q, _ = _prompt(fa, n, hk, hq, dim, page, 21, dim)
    rows = bt.expand(new, -1).contiguous()
    lens = torch.arange(n - new + 1, n + 1, dtype=torch.int32, device="cuda")
    out, lse = fa.paged_attention_lse(q[n - new:], cache, rows, lens, out_dtype=out_dtype)
    assert fa.status_query() == fa.OK
    k, v = _truth(cache, bt, n)
    qq = ref.quantized(q[n - new:].cpu())
    for i, m in enumerate(lens.tolist()):
        want, want_lse, size = ref.attend(qq[i], k[:, :m], v[:, :m])
        z = torch.einsum("hgd,hnd->hgn", qq[i].view(hk, -1, dim), k[:, :m]) / math.sqrt(dim)
        zmax = float(z.abs().max())
        bound = ref.attend_bound(want, size, m, float(v.abs().max()), zmax, out_dtype)
        assert bool(((out[i].cpu().double() - want).abs() <= bound).all()), m
        assert bool(((lse[i].cpu().double() - want_lse).abs() <= ref.lse_bound(want_lse, m, zmax)).all()), m


@pytest.mark.parametrize("batch,longest", [(257, 300), (700, 40), (1025, 200)])
def test_attention_over_more_sequences_than_one_scan(fa, cuda, batch, longest):
    """More than 256 sequences, some empty, against the 64-bit attention."""
    hk, hq, dim, page = 2, 6, 64, 16
    g = _gen(batch)
    lens = torch.randint(0, longest + 1, (batch,), generator=g)
    lens[0], lens[255:257], lens[-1] = 0, torch.tensor([longest, 0]), longest
    per_seq, pages = -(-longest // page), 400
    cache = fa.PagedCache.empty(pages, page, hk, dim)
    cache.k_codes.copy_(torch.randint(0, 256, cache.k_codes.shape, generator=g))
    cache.k_scales.copy_(torch.randint(125, 128, cache.k_scales.shape, generator=g))
    cache.v.copy_(torch.randn(cache.v.shape, generator=g))
    bt = torch.randint(0, pages, (batch, per_seq), generator=g).int()
    q = torch.randn(batch, hq, dim, generator=g).half()
    out, lse = fa.paged_attention_lse(q.cuda(), cache, bt.cuda(), lens.int().cuda(), out_dtype=F32)
    assert fa.status_query() == fa.OK
    qq, host = ref.quantized(q), (cache.k_codes.cpu(), cache.k_scales.cpu(), cache.v.cpu())
    out, lse = out.cpu().double(), lse.cpu().double()
    for b, n in enumerate(lens.tolist()):
        if n == 0:
            assert not out[b].any() and bool((lse[b] == math.inf).all())
            continue
        k, v = ref.read(host, bt[b], 0, n)
        want, want_lse, size = ref.attend(qq[b], k, v)
        z = torch.einsum("hgd,hnd->hgn", qq[b].view(hk, -1, dim), k) / math.sqrt(dim)
        zmax = float(z.abs().max())
        assert bool(((out[b] - want).abs() <= ref.attend_bound(want, size, n, float(v.abs().max()), zmax, F32)).all()), b
        assert bool(((lse[b] - want_lse).abs() <= ref.lse_bound(want_lse, n, zmax)).all()), b
