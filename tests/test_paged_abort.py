"""Paged attention when one of its waits runs out: reported, nothing written out
of place, and the next call on the same workspace right."""
import ctypes

import pytest
import torch


def test_abort_self_test_refuses_other_shapes(fa):
    """(On the host, before anything is launched.)"""
    def call(head_dim=64, q_heads=4, timeout=1000, **kw):
        D, page, heads = head_dim, 64, 1
        c = fa._serving.CacheStruct(256, 256, 256, heads * page * D // 2, heads * page * D // 32, heads * page * D * 2, 4,
                                    page, heads, D)
        return fa.lib().fp4attn_selftest_paged_abort(ctypes.byref(c), 16, 16, 1, q_heads, 16, 4, 4, 16,
                                                     kw.get("ws", 256), kw.get("wsb", 1 << 40), timeout, None)

    assert call(head_dim=128) == fa.EINVAL
    assert call(q_heads=5) == fa.EINVAL
    assert call(timeout=0) == call(timeout=10000001) == fa.EINVAL
    assert call(ws=None) == call(wsb=1) == fa.EWORKSPACE


@pytest.mark.gpu
def test_an_expired_wait_leaves_nothing_to_join(fa, cuda):
    """One sequence over every block, whose first block's waits run out.  The workspace holds what a
    call of another shape may have left there: at its start, for the join, an item of sequence 1 that
    blocks 0 to 29 share, a row that this output does not have."""
    B, hq, D, page = 5, 4, 64, 64
    g = torch.Generator().manual_seed(1)
    cache = fa.PagedCache.empty(40, page, 1, D)
    cache.k_codes.copy_(torch.randint(0, 256, cache.k_codes.shape, generator=g))
    cache.k_scales.fill_(126)
    cache.v.copy_(torch.randn(cache.v.shape, generator=g))
    blocks = 148
    n = blocks * 6 * 128  # three steps of two tiles a block
    bt = torch.randint(0, 40, (B, n // page), generator=g).int().cuda()
    q = torch.randn(B, hq, D, generator=g).half().cuda()
    ws = torch.empty(fa.paged_attention_workspace_size(cache, B, hq), dtype=torch.uint8, device="cuda")
    buf = torch.full((B, hq, D), 7.0, device="cuda")  # the calls below write its first row
    lens = torch.full((B,), n, dtype=torch.int32, device="cuda")
    one = lens[:1].clone()
    want = fa.paged_attention(q[:1], cache, bt[:1], one, out_dtype=torch.float32)
    fa.paged_attention(q, cache, bt, lens, out_dtype=torch.float32, workspace=ws)
    assert fa.status_query() == fa.OK
    for _ in range(2):
        ws[:16].view(torch.int32).copy_(torch.tensor([1, 0, 29, 1], dtype=torch.int32))
        assert fa.selftest_paged_abort(q[:1], cache, bt[:1], one, buf[:1], ws) == fa.ETIMEOUT
        assert b"device wait expired" in fa.lib().fp4attn_last_error()
        assert fa.status_query() == fa.OK
        assert bool((buf[1:] == 7).all())
        got = fa.paged_attention(q[:1], cache, bt[:1], one, out=buf[:1], workspace=ws)
        assert fa.status_query() == fa.OK and torch.equal(got, want)
        buf.fill_(7)
    # A batch of which the block that fails has the first sequence alone: the last ones have their results.
    short = torch.full((B,), n // 4, dtype=torch.int32, device="cuda")
    short[0] = n
    want = fa.paged_attention(q, cache, bt, short, out_dtype=torch.float32)
    assert fa.selftest_paged_abort(q, cache, bt, short, buf, ws) == fa.ETIMEOUT
    assert torch.equal(buf[1:], want[1:])
