"""The serving operators without a GPU: refused arguments, the rotary
frequencies, and the pages' bookkeeping."""
import ctypes
import math
import random

import pytest
import torch


# ------------------------------------------------------------- the C ABI's refusals
def _cache(fa, **kw):
    D, page, heads = kw.get("head_dim", 128), kw.get("page_size", 64), kw.get("kv_heads", 2)
    f = dict(k_codes=256, k_scales=256, v=256, k_codes_stride=heads * page * D // 2,
             k_scales_stride=heads * page * max(D // 32, 1), v_stride=heads * page * D * 2, pages=4, page_size=page,
             kv_heads=heads, head_dim=D)
    f.update(kw)
    return fa._serving.CacheStruct(*f.values())


I2, I3 = ctypes.c_int64 * 2, ctypes.c_int64 * 3


def _append(fa, cache=None, **kw):
    a = dict(K=16, V=16, Q=None, Qo=None, dt=fa.F16, tokens=2, qh=0, ks=I2(256, 128), vs=I2(256, 128), qs=None, bt=16,
             bts=4, seqs=2, maxp=4, ids=None, pos=16, table=None, rot=0, maxpos=0, inter=0, mode=0, st=None)
    a.update(kw)
    return fa.lib().fp4attn_cache_append(cache or _cache(fa), *a.values())


def _attend(fa, cache=None, **kw):
    a = dict(Q=16, O=16, lse=None, ind=fa.F16, outd=fa.F16, batch=2, qh=4, qs=I2(512, 128), bt=16, bts=4, maxp=4,
             lens=16, scale=0.0, mode=0, ws=256, wsb=1 << 40, st=None)
    a.update(kw)
    return fa.lib().fp4attn_paged_attention(cache or _cache(fa), *a.values())


def _gather(fa, cache=None, **kw):
    a = dict(bt=16, bts=4, seqs=2, maxp=4, starts=None, lens=16, most=8, heads=2, K=16, V=16, dt=fa.F16, st=None)
    a.update(kw)
    return fa.lib().fp4attn_cache_gather(cache or _cache(fa), *a.values())


def _rotary(fa, **kw):
    a = dict(x=16, y=16, dt=fa.F16, B=1, H=1, S=4, D=64, xs=I3(256, 256, 64), ys=I3(256, 256, 64), table=16, rot=64,
             maxpos=16, pos=None, ps=0, inter=0, inv=0, st=None)
    a.update(kw)
    return fa.lib().fp4attn_rotary(*a.values())


@pytest.mark.parametrize("call", ["append", "attend", "gather"])
def test_bad_caches_are_refused(fa, call):
    f = {"append": _append, "attend": _attend, "gather": _gather}[call]
    assert f(fa, _cache(fa, k_codes=None)) == fa.EINVAL
    assert f(fa, _cache(fa, head_dim=80)) == fa.EUNSUPPORTED
    for page in (0, 8, 48, 256):
        assert f(fa, _cache(fa, page_size=page)) == fa.EUNSUPPORTED
    assert f(fa, _cache(fa, pages=0)) == fa.EINVAL
    assert f(fa, _cache(fa, kv_heads=0)) == fa.EINVAL
    assert f(fa, _cache(fa, v=264)) == fa.EINVAL              # misaligned
    assert f(fa, _cache(fa, v_stride=2 * 64 * 256 - 16)) == fa.EINVAL  # less than a page
    assert f(fa, _cache(fa, k_scales_stride=520)) == fa.EINVAL  # not a multiple of 16


def test_append_refuses_bad_arguments(fa):
    assert _append(fa, dt=5) == fa.EINVAL
    assert _append(fa, mode=2) == fa.EINVAL
    assert _append(fa, tokens=-1) == fa.EINVAL
    assert _append(fa, K=None) == fa.EINVAL
    assert _append(fa, pos=None) == fa.EINVAL
    assert _append(fa, bt=None) == fa.EINVAL
    assert _append(fa, bts=3) == fa.EINVAL                      # rows shorter than max_pages
    assert _append(fa, tokens=3) == fa.EINVAL                   # three tokens, two sequences, no seq_ids
    assert b"one token per sequence" in fa.lib().fp4attn_last_error()
    assert _append(fa, Q=16) == fa.EINVAL                       # no Q_out
    assert _append(fa, Q=16, Qo=16, qh=0) == fa.EINVAL
    assert _append(fa, table=16, rot=63, maxpos=8) == fa.EINVAL
    assert _append(fa, table=16, rot=130, maxpos=8) == fa.EINVAL
    assert _append(fa, table=20, rot=64, maxpos=8) == fa.EINVAL
    assert _append(fa, table=16, rot=64, maxpos=0) == fa.EINVAL
    assert _append(fa, K=17) == fa.EINVAL
    assert _append(fa, tokens=0, ids=16, K=None) == fa.OK       # nothing to do


def test_attention_refuses_bad_arguments(fa):
    assert _attend(fa, ind=3) == fa.EINVAL
    assert _attend(fa, outd=3) == fa.EINVAL
    assert _attend(fa, mode=-1) == fa.EINVAL
    assert _attend(fa, qh=3) == fa.EINVAL                       # not a multiple of the cache's two
    assert _attend(fa, batch=-1) == fa.EINVAL
    assert _attend(fa, maxp=0) == fa.EINVAL
    assert _attend(fa, maxp=1 << 25, bts=1 << 25) == fa.EINVAL  # 2^31 tokens
    assert _attend(fa, lens=None) == fa.EINVAL
    assert _attend(fa, Q=24) == fa.EINVAL
    assert _attend(fa, qs=I2(512, 132)) == fa.EINVAL
    assert _attend(fa, ws=None) == fa.EWORKSPACE
    assert _attend(fa, wsb=1) == fa.EWORKSPACE
    assert _attend(fa, ws=128) == fa.EINVAL
    assert _attend(fa, batch=0) == fa.OK


def test_attention_workspace_size(fa):
    size = fa.lib().fp4attn_paged_attention_workspace_size
    assert size(1, 8, 8, 128) > 0
    assert size(0, 8, 8, 128) == size(1, 8, 3, 128) == size(1, 8, 8, 100) == size(1, 0, 8, 128) == 0


def test_gather_refuses_bad_arguments(fa):
    assert _gather(fa, dt=2) == fa.EINVAL
    assert _gather(fa, heads=3) == fa.EINVAL
    assert _gather(fa, most=-1) == fa.EINVAL
    assert _gather(fa, most=(1 << 30) + 1) == fa.EINVAL
    assert _gather(fa, lens=None) == fa.EINVAL
    assert _gather(fa, K=8) == fa.EINVAL
    assert _gather(fa, seqs=0) == fa.OK


def test_rotary_refuses_bad_arguments(fa):
    assert _rotary(fa, dt=2) == fa.EINVAL
    assert _rotary(fa, D=48) == fa.EUNSUPPORTED
    assert _rotary(fa, rot=0) == fa.EINVAL
    assert _rotary(fa, rot=66) == fa.EINVAL
    assert _rotary(fa, table=None) == fa.EINVAL
    assert _rotary(fa, S=17) == fa.EINVAL                       # more positions than the table has
    assert _rotary(fa, B=-1) == fa.EINVAL
    assert _rotary(fa, x=None) == fa.EINVAL
    assert _rotary(fa, y=17) == fa.EINVAL
    assert _rotary(fa, S=0) == fa.OK
    L = fa.lib()
    one = (ctypes.c_double * 1)(1.0)
    assert L.fp4attn_rotary_table(None, 1, 8, 1.0, 16, None) == fa.EINVAL
    assert L.fp4attn_rotary_table(one, 0, 8, 1.0, 16, None) == fa.EINVAL
    assert L.fp4attn_rotary_table(one, 129, 8, 1.0, 16, None) == fa.EINVAL
    assert L.fp4attn_rotary_table(one, 1, 0, 1.0, 16, None) == fa.EINVAL
    assert L.fp4attn_rotary_table((ctypes.c_double * 1)(math.nan), 1, 8, 1.0, 16, None) == fa.EINVAL
    assert L.fp4attn_rotary_table(one, 1, 8, math.inf, 16, None) == fa.EINVAL


def test_copies_refuse_bad_pages(fa):
    L = fa.lib()

    def copy(src, dst, caches=None):
        c = caches or [_cache(fa)]
        arr = (fa._serving.CacheStruct * len(c))(*c)
        i = ctypes.c_int32 * max(1, len(src))
        return L.fp4attn_copy_pages(arr, len(c), i(*src), i(*dst), len(src), None)

    assert copy([0], [4]) == fa.EINVAL                # outside
    assert copy([-1], [1]) == fa.EINVAL
    assert copy([0, 1], [2, 2]) == fa.EINVAL          # written twice
    assert b"twice" in L.fp4attn_last_error()
    assert copy([0, 1], [1, 2]) == fa.EINVAL          # read and written
    assert copy([1], [1]) == fa.EINVAL
    assert copy([3], [1], [_cache(fa), _cache(fa, pages=3)]) == fa.EINVAL  # the smallest cache counts
    assert copy([], []) == fa.OK
    assert L.fp4attn_copy_pages(None, 1, None, None, 0, None) == fa.EINVAL


# ------------------------------------------------------------- the Python wrappers' checks
def test_wrappers_refuse_tensors_off_the_gpu(fa):
    x, table = torch.zeros(1, 1, 4, 64, dtype=torch.float16), torch.zeros(4, 32, 2)
    with pytest.raises(ValueError, match="CUDA"):
        fa.rotary(x, table)
    with pytest.raises(ValueError, match="CUDA"):
        fa.PagedCache.empty(2, 16, 1, 64, device="cpu")
    with pytest.raises(ValueError, match="CUDA"):
        fa.rotary_table(4, 64, device="cpu")
    fa.copy_pages([], [0], [1])  # no caches: nothing to do


# ------------------------------------------------------------- rotary frequencies
def test_frequencies(fa):
    f, m = fa.rotary_frequencies(8, base=10000.0)
    assert m == 1.0 and f == pytest.approx([1.0, 0.1, 0.01, 0.001], rel=1e-15)
    g, m = fa.rotary_frequencies(8, scaling="linear", factor=4.0)
    assert m == 1.0 and g == pytest.approx([x / 4 for x in f], rel=1e-15)
    g, m = fa.rotary_frequencies(64, scaling="ntk", factor=4.0)
    f, _ = fa.rotary_frequencies(64)
    assert m == 1.0 and g[0] == 1.0 and g[-1] == pytest.approx(f[-1] / 4, rel=1e-12)
    assert all(a <= b for a, b in zip(g, f))


def test_yarn_keeps_fast_pairs_and_divides_slow_ones(fa):
    f, _ = fa.rotary_frequencies(128)
    g, m = fa.rotary_frequencies(128, scaling="yarn", factor=8.0, original_positions=4096)
    assert m == pytest.approx(0.1 * math.log(8.0) + 1.0)
    for a, b in zip(f, g):
        turns = 4096 * a / (2 * math.pi)
        if turns > 40:
            assert b == a
        elif turns < 0.8:
            assert b == pytest.approx(a / 8, rel=1e-12)
        else:
            assert a / 8 <= b * (1 + 1e-12) and b <= a
    # factor 1 changes nothing
    g, m = fa.rotary_frequencies(128, scaling="yarn", factor=1.0, original_positions=4096)
    assert m == 1.0 and g == pytest.approx(f, rel=1e-15)


@pytest.mark.parametrize("kw", [dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=258),
                                dict(rotary_dim=64, base=1.0), dict(rotary_dim=64, scaling="linear", factor=0.5),
                                dict(rotary_dim=64, scaling="other"), dict(rotary_dim=2, scaling="ntk", factor=2.0),
                                dict(rotary_dim=64, scaling="yarn", factor=2.0),
                                dict(rotary_dim=64, scaling="yarn", factor=2.0, original_positions=64, beta_fast=1.0)])
def test_bad_frequencies_are_refused(fa, kw):
    with pytest.raises(ValueError):
        fa.rotary_frequencies(**kw)


# ------------------------------------------------------------- pages
class _Contents:
    """What every page's tokens are, as copy_pages and appends would leave them."""

    def __init__(self, pool):
        self.pool, self.page = pool, [[None] * pool.page_size for _ in range(pool.pages)]

    def copy(self, src, dst):
        assert len(set(dst)) == len(dst) and not set(src) & set(dst)
        for s, d in zip(src, dst):
            self.page[d] = list(self.page[s])

    def append(self, seq, values):
        first = self.pool.length(seq)
        self.copy(*self.pool.extend(seq, len(values)))
        t = self.pool.table(seq)
        for i, v in enumerate(values, first):
            self.page[t[i // self.pool.page_size]][i % self.pool.page_size] = v

    def read(self, seq):
        t = self.pool.table(seq)
        return [self.page[t[i // self.pool.page_size]][i % self.pool.page_size] for i in range(self.pool.length(seq))]


@pytest.mark.parametrize("seed", range(4))
def test_pool_keeps_every_sequence_apart(fa, seed):
    rng = random.Random(seed)
    pool = fa.PagePool(40, 16)
    memory, truth, count = _Contents(pool), {}, 0
    for _ in range(600):
        seqs = list(truth)
        what = rng.choice(("new", "extend", "extend", "extend", "fork", "free", "truncate", "compact"))
        if what == "new" or not seqs:
            truth[pool.new()] = []
            continue
        seq = rng.choice(seqs)
        if what == "extend":
            n = rng.choice((0, 1, 1, 5, 16, 33))
            values = list(range(count, count + n))
            before = pool.table(seq), pool.length(seq), pool.free_pages
            try:
                memory.append(seq, values)
            except MemoryError:
                assert before == (pool.table(seq), pool.length(seq), pool.free_pages)
                continue
            truth[seq] = truth[seq] + values
            count += n
        elif what == "fork":
            truth[pool.fork(seq)] = list(truth[seq])
        elif what == "free":
            pool.free(seq)
            del truth[seq]
        elif what == "truncate":
            n = rng.randint(0, len(truth[seq]))
            pool.truncate(seq, n)
            truth[seq] = truth[seq][:n]
        else:
            memory.copy(*pool.compact())
            used = {p for s in truth for p in pool.table(s)}
            assert used == set(range(len(used)))
        for s, want in truth.items():
            assert pool.length(s) == len(want) and memory.read(s) == want
        assert pool.free_pages == 40 - len({p for s in truth for p in pool.table(s)})


def test_pool_block_tables(fa):
    pool = fa.PagePool(8, 16)
    a, b = pool.new(), pool.new()
    pool.extend(a, 40)
    t = pool.block_table([a, b])
    assert t.dtype == torch.int32 and t.tolist() == [pool.table(a), [0, 0, 0]]
    assert pool.block_table([b, a], pages=5).shape == (2, 5)
    assert pool.block_table([]).shape == (0, 1)
    with pytest.raises(ValueError):
        pool.block_table([a], pages=2)
    with pytest.raises(ValueError):
        fa.PagePool(8, 24)
    with pytest.raises(KeyError):
        pool.extend(99, 1)
    with pytest.raises(ValueError):
        pool.extend(a, -1)
    with pytest.raises(ValueError):
        pool.truncate(a, 41)
