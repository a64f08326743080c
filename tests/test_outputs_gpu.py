"""out= of the serving calls: in place, between the input's rows or apart from it,
and refused wherever its elements meet the input's or one another."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32


def _elements(base, t):
    """The elements of `base`, a flat tensor, that a view of it has, with repetitions."""
    at = torch.arange(base.numel())
    offset = (t.data_ptr() - base.data_ptr()) // base.element_size()
    return at.as_strided(t.shape, t.stride(), offset).flatten()


def test_slices_of_one_projection(fa, cuda):
    """Queries and outputs as slices of [batch, seq, heads, dim], which are not dense."""
    B, S, H, D = 2, 9, 48, 64
    qkv = torch.randn(B, S, H, D, generator=torch.Generator().manual_seed(1)).half().cuda()
    table = fa.rotary_table(S, D)

    def heads(a, b):
        return qkv[:, :, a:b].transpose(1, 2)

    for first in (1, 8, 16):
        with pytest.raises(ValueError, match="partly"):
            fa.rotary(heads(0, 32), table, out=heads(first, first + 32))
    with pytest.raises(ValueError, match="partly"):  # half of every head further
        fa.rotary(qkv[:, :, :8, :32].transpose(1, 2), fa.rotary_table(S, 32), out=qkv[:, :, :8, 16:48].transpose(1, 2))
    with pytest.raises(ValueError, match="partly"):  # the next token's rows
        fa.rotary(qkv[:, :-1].transpose(1, 2), table, out=qkv[:, 1:].transpose(1, 2))
    with pytest.raises(ValueError, match="partly"):  # the same memory, heads and tokens exchanged
        fa.rotary(qkv[:, :, :S].transpose(1, 2), table, out=qkv[:, :, :S])
    with pytest.raises(ValueError, match="share memory"):  # rows that overlap, a stride of one token's half
        fa.rotary(heads(0, 4), table, out=torch.empty(9000, dtype=F16, device="cuda").as_strided((B, 4, S, D), (4096, 1024, 32, 1)))
    want = fa.rotary(heads(0, 16), table)
    rest = qkv[:, :, 32:].clone()
    fa.rotary(heads(0, 16), table, out=heads(16, 32))       # between the input's rows
    assert torch.equal(heads(16, 32), want)
    fa.rotary(heads(0, 16), table, out=heads(0, 16))        # in place
    assert torch.equal(heads(0, 16), want) and torch.equal(qkv[:, :, 32:], rest)
    one = heads(0, 1).expand(B, 16, S, D)                   # an input that shares memory is read only
    fa.rotary(one, table, out=heads(16, 32))
    assert torch.equal(heads(16, 32), fa.rotary(one.contiguous(), table))


@pytest.mark.parametrize("seed", range(3))
def test_random_views(fa, cuda, seed):
    """Views of one buffer with strides of every kind: refused where an element is shared, else right."""
    rng = random.Random(seed)
    D, table = 32, fa.rotary_table(16, 32)
    base = torch.randn(6000, generator=torch.Generator().manual_seed(seed)).half().cuda()
    refused = done = 0
    for _ in range(300):
        shape = [rng.randint(1, 3) for _ in range(3)] + [D]

        def view():
            order, step, strides = rng.sample(range(3), 3), rng.choice((16, 32, 32, 40, 64)), [0, 0, 0]
            for k in order:
                strides[k] = step
                step = step * rng.choice((1, shape[k], shape[k], shape[k] + 1)) + rng.choice((0, 0, 8, 32))
            length = sum((n - 1) * s for n, s in zip(shape, strides)) + D
            if length > base.numel():
                return None
            return base.as_strided(shape, strides + [1], rng.randint(0, min(400, base.numel() - length)))

        x, out = view(), view()
        if rng.random() < 0.3 and x is not None and out is not None:  # the same strides, a little apart
            most = base.numel() - 1 - int(_elements(base, x).max())
            out = base.as_strided(x.shape, x.stride(), x.storage_offset() + rng.choice((0, min(most, 32), min(most, 200))))
        if x is None or out is None:
            continue
        ei, eo = _elements(base, x), _elements(base, out)
        in_place = x.data_ptr() == out.data_ptr() and all(a == b or n == 1 for a, b, n in zip(x.stride(), out.stride(), shape))
        bad = len(eo.unique()) < len(eo) or (not in_place and bool(torch.isin(ei, eo).any()))
        if bad:
            with pytest.raises(ValueError):
                fa.rotary(x, table, out=out)
            refused += 1
        else:
            want = fa.rotary(x.clone(), table)
            fa.rotary(x, table, out=out)
            assert torch.equal(out, want)
            done += 1
    assert refused > 50 and done > 50
    assert fa.status_query() == fa.OK


def test_attention_output_over_a_slice_of_queries(fa, cuda):
    """Queries inside a projection and an output in the same memory."""
    cache = fa.PagedCache.empty(4, 16, 2, 64)
    cache.k_codes.fill_(0x21), cache.k_scales.fill_(127), cache.v.normal_()
    bt, lens = torch.arange(4).int().view(2, 2).cuda(), torch.tensor([20, 32]).int().cuda()
    qkv = torch.randn(2, 8, 64, generator=torch.Generator().manual_seed(2)).half().cuda()
    q = qkv[:, :4]
    want = fa.paged_attention(q, cache, bt, lens)
    flat = qkv.view(-1)
    with pytest.raises(ValueError, match="partly"):  # contiguous, over rows of both sequences
        fa.paged_attention(q, cache, bt, lens, out=flat[256:256 + 512].view(2, 4, 64))
    with pytest.raises(ValueError, match="partly"):  # FP32 results over FP16 queries
        fa.paged_attention(qkv[:1, :4], cache, bt[:1], lens[:1], out=flat[:512].view(F32).view(1, 4, 64))
    other = torch.empty(2, 4, 64, dtype=F16, device="cuda")
    assert torch.equal(fa.paged_attention(q, cache, bt, lens, out=other), want)
    assert torch.equal(fa.paged_attention(qkv[:1, :4], cache, bt[:1], lens[:1], out=qkv[:1, 4:]), want[:1])
    assert fa.status_query() == fa.OK
