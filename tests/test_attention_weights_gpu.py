"""The weights of paged attention keep their bits: a dominating key before a long
tail of small weights, and FP16 output that differs from the 64-bit attention
by its last rounding alone."""
import math

import pytest
import torch

import serving_ref as ref

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32


def _bound(out, size, n, vmax, zmax, out_dtype):
    """How far the kernel may be off, element by element.

    Scaling a score rounds (2^-23 |z|, twice), the exponential is good to 2^-21:
    e = 2^-21 + 2^-22 |z| for every weight, 3 e for sum and quotient together;
    the FP32 sums add n / 128 + 64 roundings.  A weight w enters as two FP16
    parts, the first of 2^7 w, the second of 2^11 times what that leaves: each
    is off by 2^-11 of itself, or by half of FP16's least step, 2^-25.  Together
    2^-22 w, or 2^-25 2^-11 2^-7 = 2^-43 of the reference's weight, which the sum
    of all is not below.  Last the result is rounded to its type."""
    e = 3 * (2.0 ** -21 + 2.0 ** -22 * zmax) + (n / 128 + 64) * ref.EPS32 + 2.0 ** -22
    bound = e * size + n * 2.0 ** -43 * vmax
    if out_dtype == F16:
        return bound + ref.EPS16 * (out.abs() + bound) + 2.0 ** -25
    return bound + ref.EPS32 * out.abs()


def _check(fa, cache, q, bt, lens, out_dtype, scale):
    out, lse = fa.paged_attention_lse(q.cuda(), cache, bt.cuda(), torch.tensor(lens).int().cuda(), softmax_scale=scale,
                                      out_dtype=out_dtype)
    assert fa.status_query() == fa.OK
    qq, host = ref.quantized(q), (cache.k_codes.cpu(), cache.k_scales.cpu(), cache.v.cpu())
    for b, n in enumerate(lens):
        k, v = ref.read(host, bt[b], 0, n)
        want, want_lse, size = ref.attend(qq[b], k, v, scale)
        z = torch.einsum("hgd,hnd->hgn", qq[b].view(k.shape[0], -1, k.shape[2]), k) * scale
        zmax = float(z.abs().max())
        off, bound = (out[b].cpu().double() - want).abs(), _bound(want, size, n, float(v.abs().max()), zmax, out_dtype)
        assert bool((off <= bound).all()), (b, n, float((off / bound).max()), float((off / want.abs()).max()))
        assert bool(((lse[b].cpu().double() - want_lse).abs() <= ref.lse_bound(want_lse, n, zmax)).all())
    return out


@pytest.mark.parametrize("out_dtype", [F16, F32])
@pytest.mark.parametrize("nats", [8.0, 12.0, 17.5])
@pytest.mark.parametrize("group,dim,n", [(4, 64, 100003), (8, 128, 9001), (16, 32, 20017)])
def test_small_weights_behind_a_dominating_key(fa, cuda, group, dim, n, nats, out_dtype):
    """The first key's score lies `nats` above the others' middle and its value is zero: the
    output is the others', whose weights are small and many."""
    pages, page = 24, 64
    g = torch.Generator().manual_seed(3)
    cache = fa.PagedCache.empty(pages, page, 1, dim)
    nibble = torch.tensor([0, 0, 1, 9], dtype=torch.uint8)  # 0 and +-1/2
    pick = torch.randint(0, 4, (2,) + tuple(cache.k_codes.shape), generator=g)
    codes, v = nibble[pick[0]] | (nibble[pick[1]] << 4), torch.randn(pages, 1, page, dim, generator=g).half() + 1
    codes[0, 0, 0], v[0, 0, 0] = 0x22, 0  # 1 everywhere; a value of zero
    cache.k_codes.copy_(codes), cache.v.copy_(v)
    cache.k_scales.fill_(127)
    bt = torch.cat((torch.zeros(1), torch.randint(1, pages, (-(-n // page) - 1,), generator=g))).int()[None]
    q = torch.ones(1, group, dim, dtype=F16)
    _check(fa, cache, q, bt, [n], out_dtype, nats / dim)


@pytest.mark.parametrize("page,hk,group,dim", [(64, 2, 4, 128), (16, 2, 1, 64), (32, 1, 8, 256), (64, 1, 16, 160),
                                               (16, 1, 40, 32), (128, 2, 12, 96)])
def test_fp16_output_is_the_fp32_output_rounded(fa, cuda, page, hk, group, dim):
    g = torch.Generator().manual_seed(4)
    lens = [1, 2, 5, 127, 129, 300, 3000]
    per_seq = -(-max(lens) // page)
    cache = fa.PagedCache.empty(len(lens) * per_seq, page, hk, dim)
    cache.k_codes.copy_(torch.randint(0, 256, cache.k_codes.shape, generator=g))
    cache.k_scales.copy_(torch.randint(125, 128, cache.k_scales.shape, generator=g))
    cache.v.copy_(torch.randn(cache.v.shape, generator=g))
    bt = torch.arange(len(lens) * per_seq).int().view(len(lens), per_seq)
    q = torch.randn(len(lens), hk * group, dim, generator=g).half()
    out = [_check(fa, cache, q, bt, lens, t, 1 / math.sqrt(dim)) for t in (F16, F32)]
    assert torch.equal(out[0], out[1].half())
