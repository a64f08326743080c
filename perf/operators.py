"""What the serving operators next to the FP4 attention cost: their cases, plain forms and exact values.

The operators: rotary positions (with their gradient), the paged FP4 key / FP16 value cache (append, gather, copies
of pages) and the attention of one new token per sequence over that cache.  Keys are E2M1 codes with one UE8M0 scale
per 32 elements, as everywhere in this library; values are FP16.

`run` computes a case with elementary torch operations, or, where `own` is set, with the library's calls.
"""
import math

import torch

own = False

# Magnitudes of the E2M1 codes 0 to 7 and the borders between them (a value on a border takes the larger one).
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
BORDERS = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)


# ---------------------------------------------------------------------------------------------------------- cases
def listed():
    """The measured cases."""
    return [
        # Training on 4096-token rows: the queries of 32 heads rotated, and their gradient taken back.
        _rotary("rotary_train", batch=8, heads=32, seq=4096, dim=128, rot=128, train=True),
        # A late chunk of a long document in FP32: half of each head rotated, pairs interleaved.
        _rotary("rotary_far", batch=1, heads=16, seq=2047, dim=128, rot=64, dtype="float32", interleaved=True, first=120000),
        # Prompts entering the cache, several of unequal length at once.
        _append("append_prompts", seqs=8, new=(300, 4096), past=(0, 0), q_heads=32, kv_heads=8, dim=128, rot=128, page=64),
        # One new token for each of 16 running sequences.
        _append("append_tokens", seqs=16, new=(1, 1), past=(100, 4000), q_heads=32, kv_heads=8, dim=128, rot=128, page=64),
        # Chunks behind a cached prefix, FP32 activations, a head dimension that is no power of two, small pages.
        _append("append_chunks", seqs=3, new=(77, 700), past=(33, 1500), q_heads=16, kv_heads=16, dim=96, rot=48, page=16,
                dtype="float32", interleaved=True, ocp=True),
        # One user, a short conversation: the smallest call, where latency counts.
        _attend("attend_one", batch=1, lens=(777, 777), q_heads=32, kv_heads=8, dim=128, page=64),
        # One user, a very long document.
        _attend("attend_long", batch=1, lens=(131001, 131001), q_heads=32, kv_heads=8, dim=128, page=64),
        # A full server: many sequences of very different lengths.
        _attend("attend_batch", batch=64, lens=(1, 8192), q_heads=32, kv_heads=8, dim=128, page=64),
        # A key/value head for every query head, small pages, a small head dimension.
        _attend("attend_heads", batch=16, lens=(500, 2000), q_heads=32, kv_heads=32, dim=64, page=16),
        # Wide heads, few of them, an odd group, FP32 output.
        _attend("attend_wide", batch=8, lens=(900, 8000), q_heads=14, kv_heads=2, dim=256, page=32, out="float32", ocp=True),
        # The partly filled last page copied when 16 sequences are forked.
        _copy("pages_fork", pairs=16, pages=256, kv_heads=8, page=64, dim=128),
        # Half of a cache moved together.
        _copy("pages_compact", pairs=1500, pages=3200, kv_heads=8, page=64, dim=128),
    ]


def _named(case, name):
    return dict(case, name=name) if name else case


def _rotary(name=None, *, batch, heads, seq, dim, rot, dtype="float16", interleaved=False, first=0, train=False):
    return _named(dict(op="rotary", batch=batch, heads=heads, seq=seq, dim=dim, rot=rot, dtype=dtype,
                       interleaved=interleaved, first=first, train=train), name)


def _append(name=None, *, seqs, new, past, q_heads, kv_heads, dim, rot, page, dtype="float16", interleaved=False, ocp=False):
    return _named(dict(op="append", seqs=seqs, new_lo=new[0], new_hi=new[1], past_lo=past[0], past_hi=past[1],
                       q_heads=q_heads, kv_heads=kv_heads, dim=dim, rot=rot, page=page, dtype=dtype,
                       interleaved=interleaved, ocp=ocp), name)


def _attend(name=None, *, batch, lens, q_heads, kv_heads, dim, page, out="float16", ocp=False):
    return _named(dict(op="attend", batch=batch, len_lo=lens[0], len_hi=lens[1], q_heads=q_heads, kv_heads=kv_heads,
                       dim=dim, page=page, out=out, ocp=ocp), name)


def _copy(name=None, *, pairs, pages, kv_heads, page, dim):
    return _named(dict(op="copy", pairs=pairs, pages=pages, kv_heads=kv_heads, page=page, dim=dim), name)


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999)))))))


def draw(rng):
    """One more case of the ranges above."""
    op = rng.choice(("rotary", "append", "attend", "attend", "copy"))
    dim = rng.choice((32, 64, 96, 128, 128, 160, 256))
    page = rng.choice((16, 32, 64, 128))
    if op == "rotary":
        heads = _log_int(rng, 1, 48)
        batch = _log_int(rng, 1, 8)
        seq = _log_int(rng, 1, max(1, min(16384, (1 << 26) // (batch * heads * dim))))
        return _rotary(batch=batch, heads=heads, seq=seq, dim=dim, rot=2 * rng.randint(1, dim // 2) if rng.random() < 0.5 else dim,
                       dtype=rng.choice(("float16", "float32")), interleaved=rng.random() < 0.5,
                       first=rng.choice((0, _log_int(rng, 1, 100000))), train=rng.random() < 0.5)
    kv_heads = _log_int(rng, 1, 16)
    group = rng.choice((1, 2, 3, 4, 5, 7, 8, 8, 12, 16))
    if op == "append":
        seqs = _log_int(rng, 1, 64)
        most = max(1, min(4096, (1 << 23) // (seqs * kv_heads * dim)))
        new = (1, 1) if rng.random() < 0.4 else (1, _log_int(rng, 1, most))
        return _append(seqs=seqs, new=new, past=(0, _log_int(rng, 1, 4000)), q_heads=kv_heads * min(group, 4), kv_heads=kv_heads,
                       dim=dim, rot=2 * rng.randint(1, dim // 2) if rng.random() < 0.5 else dim, page=page,
                       dtype=rng.choice(("float16", "float32")), interleaved=rng.random() < 0.5, ocp=rng.random() < 0.5)
    if op == "attend":
        batch = _log_int(rng, 1, 100)
        longest = _log_int(rng, 1, max(1, min(100000, (1 << 27) // (batch * kv_heads * dim))))
        return _attend(batch=batch, lens=(rng.choice((0, 1, longest // 2, longest)), longest), q_heads=kv_heads * group,
                       kv_heads=kv_heads, dim=dim, page=page, out=rng.choice(("float16", "float32")), ocp=rng.random() < 0.5)
    one = kv_heads * page * (dim // 2 + dim // 32 + 2 * dim)
    pages = _log_int(rng, 4, max(4, min(4096, (1 << 29) // one)))
    return _copy(pairs=_log_int(rng, 1, pages // 2), pages=pages, kv_heads=kv_heads, page=page, dim=dim)


def _spread(n, lo, hi):
    """n lengths in [lo, hi], spread evenly, in no order; the first is hi."""
    return [lo + round((hi - lo) * (1 - (i * 0.6180339887498949) % 1.0)) for i in range(n)]


def work(case):
    """Bytes that a pass has to read and write, each once, and its operations."""
    c = case
    if c["op"] == "rotary":
        n, size = c["batch"] * c["heads"] * c["seq"] * c["dim"], 2 if c["dtype"] == "float16" else 4
        passes = 2 if c["train"] else 1
        return {"bytes": passes * (2 * n * size + c["seq"] * c["rot"] * 4), "flops": passes * n // c["dim"] * c["rot"] * 3}
    row = c["dim"] // 2 + c["dim"] // 32  # one key of one head in the cache
    if c["op"] == "append":
        tokens, size = sum(_spread(c["seqs"], c["new_lo"], c["new_hi"])), 2 if c["dtype"] == "float16" else 4
        kv, q = tokens * c["kv_heads"], tokens * c["q_heads"]
        append = kv * c["dim"] * 2 * size + kv * (row + 2 * c["dim"]) + 2 * q * c["dim"] * size + tokens * c["rot"] * 4
        gather = kv * (row + 2 * c["dim"]) + c["seqs"] * c["new_hi"] * c["kv_heads"] * c["dim"] * 4  # zeros behind a sequence's last row
        return {"bytes": append + gather, "flops": (kv + q) * c["rot"] * 3 + kv * c["dim"] * 4}
    if c["op"] == "attend":
        tokens = sum(_spread(c["batch"], c["len_lo"], c["len_hi"]))
        out = c["batch"] * c["q_heads"] * (c["dim"] * (2 + (2 if c["out"] == "float16" else 4)) + 4)
        return {"bytes": tokens * c["kv_heads"] * (row + 2 * c["dim"]) + out, "flops": 4 * tokens * c["q_heads"] * c["dim"]}
    return {"bytes": 2 * c["pairs"] * c["kv_heads"] * c["page"] * (row + 2 * c["dim"]), "flops": 0}


# --------------------------------------------------------------------------------------------------------- inputs
def _table(positions, rot, device):
    """cos and sin of position * 10000^(-2 i / rot): float32 [positions, rot / 2, 2], the angles in 64 bits."""
    freq = torch.pow(10000.0, -torch.arange(0, rot, 2, device=device, dtype=torch.float64) / rot)
    angle = torch.arange(positions, device=device, dtype=torch.float64)[:, None] * freq
    return torch.stack((angle.cos(), angle.sin()), -1).float()


def _cache(pages, kv_heads, page, dim, g, device, ocp=False):
    """A cache that holds what normal keys and values leave in it.  The reference rule scales a block's largest element
    into (1/2, 1], so its codes are 0, +-1/2 and +-1, zero most of all; the other rule (ocp) uses every code."""
    codes = torch.randint(0, 256, (pages, kv_heads, page, dim // 2), generator=g, device=device, dtype=torch.uint8)
    if not ocp:
        nibble = torch.tensor((0, 0, 0, 0, 0, 1, 1, 2, 8, 8, 8, 8, 8, 9, 9, 10), device=device, dtype=torch.uint8)
        pair = (nibble[None, :] + 16 * nibble[:, None]).flatten()
        codes = pair[codes.int()]
    low = 125 if ocp else 128
    scales = torch.randint(low, low + 2, (pages, kv_heads, page, dim // 32), generator=g, device=device, dtype=torch.uint8)
    v = torch.empty((pages, kv_heads, page, dim), device=device, dtype=torch.float16)
    v.normal_(generator=g)
    return codes, scales, v


def prepare(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    c = case
    if c["op"] == "rotary":
        # As a projection leaves it: [batch, seq, heads, dim], used as [batch, heads, seq, dim].
        shape, dtype = (c["batch"], c["seq"], c["heads"], c["dim"]), getattr(torch, c["dtype"])
        x = torch.randn(shape, generator=g, device=device, dtype=dtype).transpose(1, 2)
        positions = torch.arange(c["first"], c["first"] + c["seq"], device=device, dtype=torch.int32)
        s = {"x": x, "positions": positions, "table": _table(c["first"] + c["seq"], c["rot"], device)}
        if c["train"]:
            s["x"] = x.detach().requires_grad_()
            s["dy"] = torch.randn((c["batch"], c["heads"], c["seq"], c["dim"]), generator=g, device=device, dtype=dtype)
        return dict(s, case=c)
    if c["op"] == "append":
        new, past = _spread(c["seqs"], c["new_lo"], c["new_hi"]), _spread(c["seqs"], c["past_lo"], c["past_hi"])[::-1]
        tokens, hq, hk, dim = sum(new), c["q_heads"], c["kv_heads"], c["dim"]
        # The output of one projection for queries, keys and values, taken apart.
        qkv = torch.randn((tokens, hq + 2 * hk, dim), generator=g, device=device, dtype=getattr(torch, c["dtype"]))
        longest = max(a + b for a, b in zip(new, past))
        per_seq = -(-longest // c["page"])
        pages = c["seqs"] * per_seq + 3
        codes, scales, v = _cache(pages, hk, c["page"], dim, g, device, c["ocp"])
        block_table = torch.randperm(pages, generator=g, device=device)[: c["seqs"] * per_seq].view(c["seqs"], per_seq).int()
        counts, starts = torch.tensor(new, device=device), torch.tensor(past, device=device)
        seq_ids = torch.repeat_interleave(torch.arange(c["seqs"], device=device), counts)
        positions = torch.arange(tokens, device=device) - (counts.cumsum(0) - counts)[seq_ids] + starts[seq_ids]
        return {"case": c, "q": qkv[:, :hq], "k": qkv[:, hq : hq + hk], "v": qkv[:, hq + hk :], "k_codes": codes,
                "k_scales": scales, "v_pages": v, "block_table": block_table, "seq_ids": seq_ids.int(),
                "positions": positions.int(), "starts": starts.int(), "counts": counts.int(), "most": max(new),
                "table": _table(longest, c["rot"], device)}
    if c["op"] == "attend":
        lens = _spread(c["batch"], c["len_lo"], c["len_hi"])
        per_seq = max(1, -(-max(lens) // c["page"]))
        pages = sum(-(-n // c["page"]) for n in lens) + 2
        codes, scales, v = _cache(pages, c["kv_heads"], c["page"], c["dim"], g, device, c["ocp"])
        # Each sequence's pages, anywhere in the cache; entries behind its last page are not meant.
        order = torch.randperm(pages, generator=g, device=device)
        seq_lens = torch.tensor(lens, device=device)
        used = (seq_lens + c["page"] - 1) // c["page"]
        at = torch.arange(per_seq, device=device)[None] + (used.cumsum(0) - used)[:, None]
        block_table = torch.where(torch.arange(per_seq, device=device)[None] < used[:, None], order[at.clamp(max=pages - 1)], 0)
        q = torch.randn((c["batch"], c["q_heads"], c["dim"]), generator=g, device=device, dtype=torch.float16)
        return {"case": c, "q": q, "k_codes": codes, "k_scales": scales, "v_pages": v, "block_table": block_table.int(),
                "seq_lens": seq_lens.int()}
    codes, scales, v = _cache(c["pages"], c["kv_heads"], c["page"], c["dim"], g, device)
    order = torch.randperm(c["pages"], generator=torch.Generator().manual_seed(seed)).int()
    return {"case": c, "k_codes": codes, "k_scales": scales, "v_pages": v, "src": order[: c["pairs"]],
            "dst": order[c["pairs"] : 2 * c["pairs"]]}


# ---------------------------------------------------------------------------------------------------- plain forms
def _rotate(x, table, interleaved, inverse=False):
    """The first 2 * table.shape[-2] elements of x's last dimension (float32), as pairs, turned by their angles."""
    cos, sin = table[..., 0], -table[..., 1] if inverse else table[..., 1]
    rot = 2 * cos.shape[-1]
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = x[..., : rot // 2], x[..., rot // 2 : rot]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((turned, x[..., rot:]), -1)


def _quantize(x, ocp):
    """E2M1 codes (one per element) and scale bytes of float32 rows, one scale per 32 elements."""
    blocks = x.unflatten(-1, (-1, 32))
    top = blocks.abs().amax(-1)
    top = top / 6 if ocp else top
    m, e = torch.frexp(top)
    e = torch.where(top > 0, torch.where(m > 0.5, e, e - 1), 0)
    q = torch.ldexp(blocks, -e[..., None])
    borders = torch.tensor(BORDERS, device=x.device)
    codes = torch.bucketize(q.abs(), borders, right=True) + 8 * (q < 0)
    return codes.to(torch.uint8).flatten(-2), (e + 127).to(torch.uint8)


def _dequantize(codes, scales):
    """The float32 values of codes (one per element) with their scale bytes."""
    values = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), device=codes.device)[codes.long()]
    return torch.ldexp(values.unflatten(-1, (-1, 32)), scales.int()[..., None] - 127).flatten(-2)


def _unpack(packed):
    return torch.stack((packed & 15, packed >> 4), -1).flatten(-2)


def _read(s, positions, inside, heads_first=True):
    """Float32 keys and values [seqs, heads, length, dim] of the cache at positions [seqs, length], zero where not inside."""
    page = s["case"]["page"]
    at = s["block_table"].long().gather(1, (positions // page).clamp(0, s["block_table"].shape[1] - 1))
    off = positions % page
    k = _dequantize(_unpack(s["k_codes"][at, :, off]), s["k_scales"][at, :, off])
    v = s["v_pages"][at, :, off].float()
    k, v = (torch.where(inside[:, :, None, None], t, 0.0) for t in (k, v))
    return k.transpose(1, 2), v.transpose(1, 2)


def _plain_rotary(s):
    c, angles = s["case"], s["table"][s["positions"].long()]
    y = _rotate(s["x"].detach().float(), angles, c["interleaved"]).to(s["x"].dtype)
    if not c["train"]:
        return y
    return y, _rotate(s["dy"].float(), angles, c["interleaved"], inverse=True).to(s["x"].dtype)


def _plain_append(s):
    c, page = s["case"], s["case"]["page"]
    angles = s["table"][s["positions"].long()][:, None]
    q = _rotate(s["q"].float(), angles, c["interleaved"]).to(s["q"].dtype)
    k = _rotate(s["k"].float(), angles, c["interleaved"]).to(s["k"].dtype)
    codes, scales = _quantize(k.float(), c["ocp"])
    positions, seqs = s["positions"].long(), s["seq_ids"].long()
    at, off = s["block_table"].long()[seqs, positions // page], positions % page
    s["k_codes"][at, :, off] = codes[..., 0::2] | (codes[..., 1::2] << 4)
    s["k_scales"][at, :, off] = scales
    s["v_pages"][at, :, off] = s["v"].half()
    steps = torch.arange(s["most"], device=q.device)[None]
    k, v = _read(s, s["starts"].long()[:, None] + steps, steps < s["counts"][:, None])
    return q, k.half(), v.half()


def _plain_attend(s):
    c = s["case"]
    group = c["q_heads"] // c["kv_heads"]
    positions = torch.arange(s["block_table"].shape[1] * c["page"], device=s["q"].device)[None]
    inside = positions < s["seq_lens"][:, None]
    k, v = _read(s, positions.expand(c["batch"], -1), inside)
    q = _dequantize(*_quantize(s["q"].float(), c["ocp"])).unflatten(1, (c["kv_heads"], group))
    scores = torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(c["dim"])
    scores = scores.masked_fill(~inside[:, None, None, :], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isfinite(top), top, 0.0))
    total = p.sum(-1, keepdim=True)
    out = torch.where(total > 0, torch.matmul(p, v) / total, 0.0)
    lse = torch.where(total > 0, top + torch.log(total), math.inf)
    return out.flatten(1, 2).to(getattr(torch, c["out"])), lse.flatten(1)


def _plain_copy(s):
    src, dst = (s[n].to(s["v_pages"].device).long() for n in ("src", "dst"))
    s["k_codes"][dst] = s["k_codes"][src]
    s["k_scales"][dst] = s["k_scales"][src]
    s["v_pages"][dst] = s["v_pages"][src]
    return s["k_codes"], s["k_scales"], s["v_pages"]


# ------------------------------------------------------------------------------------------- the library's calls
def _own(s):
    import fp4attn_b200 as fa

    c = s["case"]
    if c["op"] == "rotary":
        if not c["train"]:
            return fa.rotary(s["x"], s["table"], s["positions"], interleaved=c["interleaved"])
        y = fa.rotary_embedding(s["x"], s["table"], s["positions"], interleaved=c["interleaved"])
        return y.detach(), torch.autograd.grad(y, s["x"], s["dy"])[0]
    # The handle of the cache, which a program makes once.
    cache = s.get("cache")
    if cache is None:
        cache = s["cache"] = fa.PagedCache(s["k_codes"], s["k_scales"], s["v_pages"])
    rule = "ocp" if c.get("ocp") else "reference"
    if c["op"] == "append":
        q = fa.cache_append(cache, s["k"], s["v"], s["block_table"], s["positions"], s["seq_ids"], Q=s["q"],
                            table=s["table"], interleaved=c["interleaved"], scale_mode=rule)
        return (q, *fa.cache_gather(cache, s["block_table"], s["starts"], s["counts"], s["most"]))
    if c["op"] == "attend":
        if "workspace" not in s:
            size = fa.paged_attention_workspace_size(cache, c["batch"], c["q_heads"])
            s["workspace"] = torch.empty(size, dtype=torch.uint8, device=s["q"].device)
        return fa.paged_attention_lse(s["q"], cache, s["block_table"], s["seq_lens"], out_dtype=getattr(torch, c["out"]),
                                      scale_mode=rule, workspace=s["workspace"])
    fa.copy_pages([cache], s["src"], s["dst"])
    return s["k_codes"], s["k_scales"], s["v_pages"]


def run(state):
    """One pass: rotary y (and dx); append (rotated queries, the new keys and values read back out of the cache);
    attend (out, log-sum-exp); copy (the cache: bytes, copied as they are)."""
    if own:
        return _own(state)
    return {"rotary": _plain_rotary, "append": _plain_append, "attend": _plain_attend, "copy": _plain_copy}[state["case"]["op"]](state)


# ---------------------------------------------------------------------------------------------------------- exact
def _turned(x, table, interleaved, sign=1.0):
    """x in 64 bits, as complex numbers times the table's: conjugated for the gradient."""
    rot = 2 * table.shape[-2]
    x = x.double()
    pairs = x[..., :rot].unflatten(-1, (-1, 2) if interleaved else (2, -1))
    if not interleaved:
        pairs = pairs.transpose(-1, -2)
    turn = torch.complex(table[..., 0].double(), sign * table[..., 1].double())
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    if not interleaved:
        z = z.transpose(-1, -2)
    return torch.cat((z.flatten(-2), x[..., rot:]), -1)


def _nearest(x, ocp):
    """Every element of 64-bit rows as the multiple of its block's scale that the 4-bit type has nearest to it."""
    b = x.unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True) / (6.0 if ocp else 1.0)
    scale = torch.where(top > 0, torch.exp2(torch.ceil(torch.log2(torch.where(top > 0, top, 1.0)))), 1.0)
    a = (b / scale).abs()
    # Steps of 1/2 below 2, of 1 from 2 to 4, of 2 above; half a step rounds up; 6 is the largest.
    step = torch.where(a < 1.75, 0.5, torch.where(a < 3.5, 1.0, 2.0)).double()
    return (torch.sign(b) * torch.clamp(torch.floor(a / step + 0.5) * step, max=6.0) * scale).flatten(-2)


def _values(packed, scales):
    """64-bit values of packed codes from the bits of each: sign, two of exponent, one of fraction."""
    n = torch.stack((packed % 16, packed // 16), -1).flatten(-2).int()
    exponent, fraction = (n // 2) % 4, (n % 2).double()
    a = torch.where(exponent == 0, fraction / 2, (1 + fraction / 2) * torch.exp2(exponent.double() - 1))
    a = torch.where(n >= 8, -a, a)
    return (a.unflatten(-1, (-1, 32)) * torch.exp2(scales.double() - 127)[..., None]).flatten(-2)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "rotary":
        angles = s["table"][s["positions"].long()]
        y = _turned(s["x"].detach(), angles, c["interleaved"])
        return (y, _turned(s["dy"], angles, c["interleaved"], -1.0)) if c["train"] else y
    if c["op"] == "append":
        angles = s["table"][s["positions"].long()][:, None]
        q = _turned(s["q"], angles, c["interleaved"])
        # A key is rounded to its type before it is quantised, as it is where rotating and quantising are two steps.
        k = _nearest(_turned(s["k"], angles, c["interleaved"]).to(s["k"].dtype).double(), c["ocp"])
        out = torch.zeros((2, c["seqs"], c["kv_heads"], s["most"], c["dim"]), dtype=torch.float64, device=q.device)
        first = 0
        for i, n in enumerate(s["counts"].tolist()):
            out[0, i, :, :n] = k[first : first + n].transpose(0, 1)
            out[1, i, :, :n] = s["v"][first : first + n].double().transpose(0, 1)
            first += n
        return q, out[0], out[1]
    if c["op"] == "attend":
        q = _nearest(s["q"].double(), c["ocp"])
        out = torch.zeros((c["batch"], c["q_heads"], c["dim"]), dtype=torch.float64, device=q.device)
        lse = torch.full((c["batch"], c["q_heads"]), math.inf, dtype=torch.float64, device=q.device)
        group = c["q_heads"] // c["kv_heads"]
        for i, n in enumerate(s["seq_lens"].tolist()):
            if n == 0:
                continue
            pages = s["block_table"][i, : -(-n // c["page"])].long()
            for h in range(c["kv_heads"]):
                heads = slice(h * group, (h + 1) * group)
                k = _values(s["k_codes"][pages, h], s["k_scales"][pages, h]).flatten(0, 1)[:n]
                z = q[i, heads] @ k.T / math.sqrt(c["dim"])
                lse[i, heads] = torch.logsumexp(z, -1)
                out[i, heads] = torch.softmax(z, -1) @ s["v_pages"][pages, h].flatten(0, 1)[:n].double()
        return out, lse
    v = s["v_pages"].double()
    v[s["dst"].to(v.device).long()] = v[s["src"].to(v.device).long()]
    return None, None, v
