"""Measured cases of the paged 8-bit KV cache and the operators around it.

Four operators, as a generation loop uses them:

  norm_rope   per-head RMS norm of queries and keys with the rotary embedding in the same pass
  append      the new rows of a step or a prefill: norm + rotation of q / k, then K and V quantised to 8 bits
              into the pages of the cache; the rows just written are read back (what a caller that hands them
              to another operator does)
  read        reading a range of cached positions back as fp32 rows
  attn        attention of a chunk of new rows (one token .. thousands) over the paged cache

A cache row of one head holds 8-bit codes and one power-of-two exponent e: value = code * 2^e, with e the least
integer for which max|x| <= Qmax * 2^e (Qmax = 127 for int8, 448 for e4m3) and the code rounded to nearest even.
"""
import math

import torch

own = False

DEV = "cuda"
EPS = 1e-6
QMAX = {"int8": 127.0, "e4m3": 448.0}
EMIN = {"int8": -126, "e4m3": -117}


# ------------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # one decode step of eight sequences: the smallest launch, pure latency
        dict(name="norm_rope_step", op="norm_rope", rows=8, heads=16, kv_heads=4, hd=64),
        # a prefill's projection rows, grouped heads of 128
        dict(name="norm_rope_prefill", op="norm_rope", rows=16384, heads=32, kv_heads=8, hd=128),
        # one new token for each of 64 sequences
        dict(name="append_step", op="append", fmt="e4m3", batch=64, heads=16, kv_heads=8, hd=64, page=16, new=1,
             ragged=False, lo=64, hi=1024),
        # block verify: four drafted rows for each of 2048 sequences
        dict(name="append_verify", op="append", fmt="int8", batch=2048, heads=16, kv_heads=4, hd=64, page=32, new=4,
             ragged=False, lo=64, hi=512),
        # ragged prefill of 24 prompts
        dict(name="append_prefill", op="append", fmt="e4m3", batch=24, heads=32, kv_heads=8, hd=128, page=64, new=2501,
             ragged=True, lo=0, hi=700),
        # a short prefix handed to an operator that wants fp32 rows
        dict(name="read_prefix", op="read", fmt="int8", batch=4, kv_heads=4, hd=64, page=16, lo=96, hi=513),
        # whole caches of a batch
        dict(name="read_caches", op="read", fmt="e4m3", batch=48, kv_heads=8, hd=128, page=48, lo=1000, hi=4099),
        # one token of two short sequences of a small byte decoder
        dict(name="attn_token_small", op="attn", fmt="e4m3", batch=2, heads=4, kv_heads=4, hd=64, page=16, new=1,
             ragged=False, lo=200, hi=513, window=0, block=False),
        # one token of many sequences, a head of keys for every head of queries
        dict(name="attn_token_batch", op="attn", fmt="int8", batch=256, heads=16, kv_heads=16, hd=64, page=32, new=1,
             ragged=False, lo=64, hi=4096, window=0, block=False),
        # drafted blocks over long caches, grouped heads
        dict(name="attn_block_verify", op="attn", fmt="e4m3", batch=64, heads=32, kv_heads=8, hd=128, page=64, new=8,
             ragged=False, lo=1500, hi=8191, window=0, block=True),
        # a chunk of a long prompt
        dict(name="attn_chunk_long", op="attn", fmt="e4m3", batch=1, heads=16, kv_heads=4, hd=64, page=64, new=2048,
             ragged=False, lo=30001, hi=30001, window=0, block=False),
        # chunks of eight prompts at different places, a window, pages of an odd size
        dict(name="attn_chunk_ragged", op="attn", fmt="int8", batch=8, heads=16, kv_heads=8, hd=128, page=48, new=1021,
             ragged=True, lo=0, hi=8100, window=4000, block=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["norm_rope", "append", "read", "attn", "attn", "attn"])
    hd = rng.choice([32, 64, 64, 128])
    kv = rng.choice([1, 2, 4, 8, 16])
    heads = kv * rng.choice([g for g in (1, 2, 4, 8) if kv * g <= 32])
    fmt, page = rng.choice(["int8", "e4m3"]), 16 * _log(rng, 1, 8)
    if op == "norm_rope":
        c = dict(op=op, rows=_log(rng, 1, 20000), heads=heads, kv_heads=kv, hd=hd)
        while _cost(c) > _cost(listed()[1]):
            c["rows"] //= 2
        return c
    if op == "append":
        c = dict(op=op, fmt=fmt, batch=_log(rng, 1, 512), heads=heads, kv_heads=kv, hd=hd, page=page,
                 new=_log(rng, 1, 2501), ragged=rng.random() < 0.5, lo=rng.choice([0, 17]), hi=_log(rng, 20, 1024))
        while _cost(c) > _cost(listed()[4]):
            c["batch" if c["batch"] > 1 else "new"] //= 2
        return c
    if op == "read":
        c = dict(op=op, fmt=fmt, batch=_log(rng, 1, 64), kv_heads=kv, hd=hd, page=page, lo=rng.choice([0, 1, 33]),
                 hi=_log(rng, 40, 4099))
        while _cost(c) > _cost(listed()[6]):
            c["batch"] //= 2
        return c
    if rng.random() < 0.5:  # one token, or a drafted block
        c = dict(op=op, fmt=fmt, batch=_log(rng, 1, 256), heads=heads, kv_heads=kv, hd=hd, page=page,
                 new=rng.choice([1, 1, 1, 2, 3, 5, 8, 17]), ragged=False, lo=rng.choice([0, 63]), hi=_log(rng, 64, 8191),
                 window=rng.choice([0, 0, 500]), block=rng.random() < 0.3)
        big = listed()[9]
    else:  # a chunk
        c = dict(op=op, fmt=fmt, batch=_log(rng, 1, 12), heads=heads, kv_heads=kv, hd=hd, page=page,
                 new=_log(rng, 18, 2048), ragged=rng.random() < 0.5, lo=rng.choice([0, 100]), hi=_log(rng, 128, 16000),
                 window=rng.choice([0, 0, 1000]), block=False)
        big = listed()[10]
    while _cost(c) > _cost(big) or c["batch"] * c["heads"] * c["new"] * (c["hi"] + c["new"]) > 1.2e9:
        c["batch" if c["batch"] > 1 else "hi" if c["hi"] > 200 else "new"] //= 2
        c["lo"] = min(c["lo"], c["hi"])
    return c


def _spread(n, lo, hi, phase):
    """n whole numbers over [lo, hi], in no order: the same for everybody."""
    if n == 1:
        return [hi]
    return [lo + int((hi - lo) * ((0.6180339887498949 * i + phase) % 1.0) + 0.5) for i in range(n)]


def _new(case):
    """New rows of each sequence; a ragged batch has one without any."""
    if not case["ragged"]:
        return [case["new"]] * case["batch"]
    n = _spread(case["batch"], 1, case["new"], 0.37)
    if len(n) > 2:
        n[1] = 0
    n[0] = case["new"]
    return n


def _base(case):
    return _spread(case["batch"], case["lo"], case["hi"], 0.11)


def _pairs(case):
    """(query, key) pairs that a mask leaves, and keys that some query sees, over the batch."""
    pairs = keys = 0
    for b, n in zip(_base(case), _new(case)):
        if n == 0:
            continue
        if case["block"]:
            pairs, keys = pairs + n * (b + n), keys + b + n
            continue
        w = case["window"] or 1 << 40
        full = max(0, min(n, w - b))  # rows that see everything up to themselves: b + 1 .. b + full keys
        pairs += full * b + full * (full + 1) // 2 + (n - full) * w
        keys += min(b + n, w + n - 1)
    return pairs, keys


def work(case):
    hd, kv = case["hd"], case["kv_heads"]
    if case["op"] == "norm_rope":
        values = case["rows"] * (case["heads"] + kv) * hd
        return {"bytes": 8 * values + 4 * hd * (case["rows"] + 2), "flops": 8 * values}
    if case["op"] == "append":
        rows, H = sum(_new(case)), case["heads"]
        return {"bytes": rows * hd * (8 * H + 8 * kv) + rows * 2 * kv * (hd + 1) + rows * 2 * kv * hd * 2 + rows * hd * 4,
                "flops": rows * hd * (8 * H + 14 * kv)}
    if case["op"] == "read":
        rows = sum(_base(case))
        return {"bytes": rows * 2 * kv * (hd + 1 + 4 * hd), "flops": rows * 2 * kv * hd}
    pairs, keys = _pairs(case)
    return {"bytes": keys * 2 * kv * (hd + 1) + 8 * sum(_new(case)) * case["heads"] * hd,
            "flops": 4 * hd * case["heads"] * pairs}


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 6.5e12, w["flops"] / 4e14)


# ------------------------------------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 11)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)


def _tables(positions, hd):
    """cos / sin [positions, hd / 2], rounded once from 64 bits."""
    freq = 10000.0 ** (-torch.arange(0, hd, 2, device=DEV, dtype=torch.float64) / hd)
    a = torch.arange(positions, device=DEV, dtype=torch.float64)[:, None] * freq[None, :]
    return a.cos().float(), a.sin().float()


def _cu(lens):
    return torch.tensor([0] + lens, device=DEV).cumsum(0).to(torch.int32)


def _ints(v):
    return torch.tensor(v, device=DEV, dtype=torch.int32)


def _pages(g, case, lens):
    """A page table whose pages lie in no order, for lens[b] positions of each sequence; pages beyond them are -1."""
    need = [-(-n // case["page"]) for n in lens]
    most, total = max(max(need), 1), sum(need) + 3
    order = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
    first = torch.tensor([0] + need, device=DEV).cumsum(0)[:-1]
    at = torch.arange(most, device=DEV)[None, :]
    table = order[(first[:, None] + at).clamp(max=total - 1)]
    return torch.where(at < torch.tensor(need, device=DEV)[:, None], table, -1).contiguous(), total


def _filled(g, case, lens):
    """A cache that holds rows already: codes and exponents of normal values, of a different size for each head."""
    table, total = _pages(g, case, lens)
    s = dict(page_table=table)
    for n in ("k", "v"):
        x = _normal(g, total, case["kv_heads"], case["page"], case["hd"])
        x *= torch.exp2(torch.rand(1, case["kv_heads"], 1, 1, generator=g, device=DEV) * 2 - 1)
        s[n + "_codes"], s[n + "_exp"] = _quantise(x, case["fmt"])
        del x
    return s


def prepare(case, seed):
    g = _gen(seed)
    hd, s = case["hd"], dict(case=dict(case))
    if case["op"] == "norm_rope":
        H, kv, rows = case["heads"], case["kv_heads"], case["rows"]
        qkv = _normal(g, rows, (H + 2 * kv) * hd)  # the packed projection: q and k are read in place
        s.update(q=qkv[:, :H * hd], k=qkv[:, H * hd:(H + kv) * hd], qkv=qkv)
        s["pos"] = torch.randint(0, 8192, (rows,), generator=g, device=DEV, dtype=torch.int32)
        s["q_gain"], s["k_gain"] = (1 + 0.2 * _normal(g, hd) for _ in range(2))
        s["cos"], s["sin"] = _tables(8192, hd)
        s["q_out"], s["k_out"] = (torch.empty(rows, n * hd, device=DEV) for n in (H, kv))
        return s
    if case["op"] == "append":
        H, kv, new, base = case["heads"], case["kv_heads"], _new(case), _base(case)
        rows = sum(new)
        qkv = _normal(g, rows, (H + 2 * kv) * hd)
        s.update(q=qkv[:, :H * hd], k=qkv[:, H * hd:(H + kv) * hd], v=qkv[:, (H + kv) * hd:], qkv=qkv)
        s["q_gain"], s["k_gain"] = (1 + 0.2 * _normal(g, hd) for _ in range(2))
        s["cos"], s["sin"] = _tables(max(b + n for b, n in zip(base, new)) + 1, hd)
        s["page_table"], total = _pages(g, case, [b + n for b, n in zip(base, new)])
        for n in ("k", "v"):
            s[n + "_codes"] = torch.zeros(total, kv, case["page"], hd, device=DEV, dtype=torch.uint8)
            s[n + "_exp"] = torch.zeros(total, kv, case["page"], device=DEV, dtype=torch.int8)
            s[n + "_back"] = torch.empty(rows, kv * hd, device=DEV, dtype=torch.bfloat16)
        s["cu_new"], s["base_len"] = _cu(new), _ints(base)
        s["q_out"] = torch.empty(rows, H * hd, device=DEV)
        s["max_new"] = max(new)
        return s
    if case["op"] == "read":
        lens = _base(case)
        s.update(_filled(g, case, lens))
        s["cu_rows"] = _cu(lens)
        for n in ("k", "v"):
            s[n + "_out"] = torch.empty(sum(lens), case["kv_heads"] * hd, device=DEV)
        return s
    new, base = _new(case), _base(case)
    s.update(_filled(g, case, [b + n for b, n in zip(base, new)]))
    s["cu_new"], s["base_len"] = _cu(new), _ints(base)
    s["q"] = _normal(g, sum(new), case["heads"] * hd)
    s["out"] = torch.empty_like(s["q"])
    s["max_new"], s["max_len"] = max(new), max(b + n for b, n in zip(base, new))
    return s


# ------------------------------------------------------------------------------------------------ plain form

def _quantise(x, fmt):
    """Codes (as bytes) and exponents of rows x [..., hd]."""
    m, e = torch.frexp(x.abs().amax(-1))
    if fmt == "int8":
        e = torch.where(m <= 127 / 128, e - 7, e - 6).clamp(-126, 121)
    else:
        e = torch.where(m <= 0.875, e - 9, e - 8).clamp(-117, 119)
    y = torch.ldexp(x, -e[..., None])
    if fmt == "int8":
        return y.round_().clamp_(-127, 127).to(torch.int8).view(torch.uint8), e.to(torch.int8)
    return y.clamp_(-448, 448).float().to(torch.float8_e4m3fn).view(torch.uint8), e.to(torch.int8)


def _values(codes, exp, fmt):
    x = codes.view(torch.int8 if fmt == "int8" else torch.float8_e4m3fn).float()
    return x * torch.exp2(exp.float())[..., None]


def _norm_rope(x, heads, hd, gain, cos, sin, pos):
    """[rows, heads, hd] in 64 bits: what is quantised next may lie beside a border."""
    x = x.double().reshape(-1, heads, hd)
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * gain.double()
    c, s = cos.double()[pos.long()][:, None, :], sin.double()[pos.long()][:, None, :]
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)


def _row_owner(cu, rows):
    """(sequence, index in it) of every packed row."""
    r = torch.arange(rows, device=DEV)
    b = torch.searchsorted(cu[1:].long(), r, right=True)
    return b, r - cu.long()[b]


def _plain_norm_rope(s):
    c = s["case"]
    hd = c["hd"]
    q = _norm_rope(s["q"], c["heads"], hd, s["q_gain"], s["cos"], s["sin"], s["pos"])
    k = _norm_rope(s["k"], c["kv_heads"], hd, s["k_gain"], s["cos"], s["sin"], s["pos"])
    return {"q": q.float().flatten(1), "k": k.float().flatten(1)}


def _plain_append(s):
    c = s["case"]
    hd, kv = c["hd"], c["kv_heads"]
    b, i = _row_owner(s["cu_new"], s["q"].shape[0])
    pos = s["base_len"].long()[b] + i
    q = _norm_rope(s["q"], c["heads"], hd, s["q_gain"], s["cos"], s["sin"], pos)
    k = _norm_rope(s["k"], kv, hd, s["k_gain"], s["cos"], s["sin"], pos)
    v = s["v"].reshape(-1, kv, hd)
    page, slot = s["page_table"].long()[b, pos // c["page"]], pos % c["page"]
    back = {}
    for n, x in (("k", k), ("v", v)):
        s[n + "_codes"][page, :, slot], s[n + "_exp"][page, :, slot] = _quantise(x, c["fmt"])
        x = _values(s[n + "_codes"][page, :, slot], s[n + "_exp"][page, :, slot], c["fmt"])
        back[n] = x.to(torch.bfloat16).flatten(1)
    return {"q": q.float().flatten(1), "k": back["k"], "v": back["v"]}


def _plain_read(s):
    c = s["case"]
    b, i = _row_owner(s["cu_rows"], s["k_out"].shape[0])
    page, slot = s["page_table"].long()[b, i // c["page"]], i % c["page"]
    k, v = (_values(s[n + "_codes"][page, :, slot], s[n + "_exp"][page, :, slot], c["fmt"]).flatten(1) for n in ("k", "v"))
    return {"k": k, "v": v}


def _plain_attn(s):
    c = s["case"]
    B, H, kv, hd = c["batch"], c["heads"], c["kv_heads"], c["hd"]
    n, L, G = s["max_new"], s["max_len"], H // kv
    cu, base = s["cu_new"].long(), s["base_len"].long()
    new = cu[1:] - cu[:-1]
    table = s["page_table"].long().clamp(min=0)
    k, v = (_values(s[m + "_codes"][table], s[m + "_exp"][table], c["fmt"]) for m in ("k", "v"))
    k, v = (x.transpose(1, 2).reshape(B, kv, -1, hd)[:, :, :L] for x in (k, v))  # pages side by side
    i, j = torch.arange(n, device=DEV), torch.arange(L, device=DEV)
    p = base[:, None] + i[None, :]
    ok = (j[None, None, :] < (base + new)[:, None, None]) & (i[None, :, None] < new[:, None, None])
    if not c["block"]:
        ok = ok & (j[None, None, :] <= p[:, :, None])
        if c["window"]:
            ok = ok & (p[:, :, None] - j[None, None, :] < c["window"])
    rows = (cu[:-1, None] + i[None, :]).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][rows].reshape(B, n, kv, G, hd).permute(0, 2, 3, 1, 4).reshape(B, kv, G * n, hd)
    x = torch.matmul(q, k.transpose(-1, -2)) * (1 / math.sqrt(hd))
    x = x.view(B, kv, G, n, L).masked_fill_(~ok[:, None, None], -math.inf)
    m = x.amax(-1, keepdim=True).clamp(min=-1e30)
    x = x.sub_(m).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(B, kv, G * n, L), v).view(B, kv, G, n, hd) / total.clamp(min=1e-30)
    o = o.permute(0, 3, 1, 2, 4).reshape(B, n, H * hd)
    live = i[None, :] < new[:, None]
    return {"out": o[live]}


# ------------------------------------------------------------------------------------------------ one pass

def _cache(s):
    from fblt_b200 import ops
    c = s["case"]
    return ops.PagedKvCache(s["k_codes"], s["v_codes"], s["k_exp"], s["v_exp"], s["page_table"], c["fmt"])


def _plan(s):
    """The descriptors (and the workspace) that a program makes once for its buffers and keeps."""
    from fblt_b200 import ops
    c = s["case"]
    if c["op"] == "norm_rope":
        return ops.make_qk_norm_rope(s["q"], s["k"], s["pos"], c["heads"], c["kv_heads"], c["hd"], q_out=s["q_out"],
                                     k_out=s["k_out"], q_gain=s["q_gain"], k_gain=s["k_gain"], eps=EPS,
                                     rope_cos=s["cos"], rope_sin=s["sin"])
    cache = _cache(s)
    if c["op"] == "append":
        return (ops.make_paged_append(cache, s["cu_new"], s["base_len"], s["k"], s["v"], q=s["q"], q_out=s["q_out"],
                                      num_heads=c["heads"], q_gain=s["q_gain"], k_gain=s["k_gain"], eps=EPS,
                                      rope_cos=s["cos"], rope_sin=s["sin"]),
                ops.make_paged_read(cache, s["cu_new"], s["k_back"], s["v_back"], start=s["base_len"]))
    if c["op"] == "read":
        return ops.make_paged_read(cache, s["cu_rows"], s["k_out"], s["v_out"])
    d = ops.make_paged_attn(cache, s["cu_new"], s["base_len"], s["q"], s["out"], c["heads"], s["max_new"], s["max_len"],
                            1 / math.sqrt(c["hd"]), block_mode=c["block"], window=c["window"])
    return d, ops.paged_attn_workspace(d)


def _own(s):
    from fblt_b200 import ops
    if "plan" not in s:
        s["plan"] = _plan(s)
    op, plan = s["case"]["op"], s["plan"]
    if op == "norm_rope":
        ops.qk_norm_rope(plan)
        return {"q": s["q_out"], "k": s["k_out"]}
    if op == "append":
        ops.paged_append(plan[0])
        ops.paged_read(plan[1])
        return {"q": s["q_out"], "k": s["k_back"], "v": s["v_back"]}
    if op == "read":
        ops.paged_read(plan)
        return {"k": s["k_out"], "v": s["v_out"]}
    ops.paged_attn(*plan)
    return {"out": s["out"]}


def run(s):
    if own:
        return _own(s)
    op = s["case"]["op"]
    return {"norm_rope": _plain_norm_rope, "append": _plain_append, "read": _plain_read, "attn": _plain_attn}[op](s)


# ------------------------------------------------------------------------------------------------ in 64 bits

def _exact_rows(x, heads, hd, gain, cos, sin, pos):
    """Norm and rotation by the definition, with complex numbers for the pairs."""
    x = x.double().reshape(x.shape[0], heads, hd)
    y = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / hd + EPS) * gain.double()
    turn = torch.complex(cos.double()[pos], sin.double()[pos])[:, None, :]
    z = torch.view_as_complex(y.reshape(y.shape[0], heads, hd // 2, 2).contiguous()) * turn
    return torch.view_as_real(z).reshape(y.shape[0], heads, hd)


def _exact_stored(x, fmt):
    """The values that codes and exponent of rows x stand for, by logarithm and grid."""
    q = QMAX[fmt]
    a = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(a / q))
    e = torch.where(a > q * torch.exp2(e), e + 1, torch.where(a <= q * torch.exp2(e - 1), e - 1, e)).clamp(min=EMIN[fmt])
    y = x * torch.exp2(-e)
    if fmt == "int8":
        y = torch.round(y)
    else:  # three bits behind the leading one, a fixed grid below 2^-6
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
        y = torch.round(y / step) * step
    return y * torch.exp2(e)


def exact(case, seed):
    s = prepare(case, seed)
    hd = case["hd"]
    if case["op"] == "norm_rope":
        pos = s["pos"].long()
        return {"q": _exact_rows(s["q"], case["heads"], hd, s["q_gain"], s["cos"], s["sin"], pos).flatten(1),
                "k": _exact_rows(s["k"], case["kv_heads"], hd, s["k_gain"], s["cos"], s["sin"], pos).flatten(1)}
    kv = case["kv_heads"]
    if case["op"] == "append":
        pos = torch.cat([torch.arange(b, b + n, device=DEV) for b, n in zip(_base(case), _new(case))])
        q = _exact_rows(s["q"], case["heads"], hd, s["q_gain"], s["cos"], s["sin"], pos)
        k = _exact_rows(s["k"], kv, hd, s["k_gain"], s["cos"], s["sin"], pos)
        v = s["v"].double().reshape(-1, kv, hd)
        return {"q": q.flatten(1), "k": _exact_stored(k, case["fmt"]).flatten(1), "v": _exact_stored(v, case["fmt"]).flatten(1)}

    def rows_of(name, b, n):
        """Positions 0 .. n of sequence b: [kv_heads, n, hd]."""
        at = s["page_table"][b, :-(-n // case["page"])].long()
        code = s[name + "_codes"][at].view(torch.int8 if case["fmt"] == "int8" else torch.float8_e4m3fn)
        x = code.float().double() * 2.0 ** s[name + "_exp"][at].double()[..., None]
        return x.permute(1, 0, 2, 3).reshape(kv, -1, hd)[:, :n]

    if case["op"] == "read":
        return {n: torch.cat([rows_of(n, b, m).transpose(0, 1).flatten(1) for b, m in enumerate(_base(case))]) for n in ("k", "v")}
    H, out, at = case["heads"], torch.empty(s["q"].shape, device=DEV, dtype=torch.float64), 0
    for b, (base, n) in enumerate(zip(_base(case), _new(case))):
        k, v = rows_of("k", b, base + n), rows_of("v", b, base + n)
        key = torch.arange(base + n, device=DEV)
        step = max(1, (1 << 28) // (H * (base + n)))
        for i in range(0, n, step):
            m = min(step, n - i)
            q = s["q"][at + i:at + i + m].double().reshape(m, kv, H // kv, hd)
            x = torch.einsum("ihgd,hkd->hgik", q, k) / math.sqrt(hd)
            gap = (base + i + torch.arange(m, device=DEV))[:, None] - key[None, :]
            if not case["block"]:
                x = x.masked_fill((gap < 0) | ((gap >= case["window"]) if case["window"] else False), -math.inf)
            out[at + i:at + i + m] = torch.einsum("hgik,hkd->ihgd", torch.softmax(x, -1), v).reshape(m, H * hd)
            del x
        at += n
    return {"out": out}
