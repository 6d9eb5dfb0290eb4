"""Workloads of the K/V cache operators and of shared-prefix attention, for timing and comparing.

Three operators of a serving loop over a paged K/V cache:

  shared_prefix   one query token per sequence over a prefix that all sequences of the batch share, followed by each
                  sequence's own tokens (packed, or in pages): decoding_attn_shared_prefix_fwd and
                  decoding_attn_paged_shared_prefix_fwd
  append          the new K/V rows of every sequence quantised as they are written into the page pools, and read back:
                  kv_cache_append, kv_cache_read (a 16-bit cache: written only; the pools are the result)
  read            whole sequences gathered out of the page pools and de-quantised: kv_cache_read

`run` computes them in their plain form (elementary torch operations), or, where `own` is true, through this package.

What an append stores, in 64-bit arithmetic, s, scale and zero being float32 values:
  fp8 / int8 / int4 with a factor s per KV head:  the nearest e4m3 number (ties to even, at most +-448 in magnitude), or the
      nearest integer (ties to even, clamped to the type's range), of x / s
  *_tok (a pair per row), *_g64 (a pair per 64 elements of a row): scale = (max - min) / (2^bits - 1), at least 1e-8,
      zero = qmin - min / scale, n = the nearest integer to x / scale + zero (ties to even, clamped)
and what a read returns: s n, or scale (n - zero).
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_QMIN = {"int8": -128, "int4": -8}
_QMAX = {"int8": 127, "int4": 7}


def listed():
    return [
        # a few chats behind a short system prompt: nothing but latency
        dict(name="prefix_small", op="shared_prefix", dtype="bf16", batch=4, head_q=32, head_k=8, dim=128, prefix=256,
             own=32, page=0, alibi=False, padded=0),
        # an ordinary serving step: 64 chats behind one system prompt with examples, a paged cache, a padded batch
        dict(name="prefix_gqa_paged", op="shared_prefix", dtype="bf16", batch=64, head_q=32, head_k=8, dim=128,
             prefix=4096, own=1024, page=16, alibi=False, padded=3),
        # many samples of one long document's question: the largest
        dict(name="prefix_gqa_long", op="shared_prefix", dtype="bf16", batch=256, head_q=32, head_k=8, dim=128,
             prefix=16384, own=1024, page=0, alibi=False, padded=0),
        # every head with K/V of its own, positions by ALiBi, odd lengths
        dict(name="prefix_mha_alibi", op="shared_prefix", dtype="fp16", batch=96, head_q=32, head_k=32, dim=64,
             prefix=1000, own=257, page=0, alibi=True, padded=0),
        # one KV head for all query heads, wide heads, candidates that have just begun to differ
        dict(name="prefix_mqa_wide", op="shared_prefix", dtype="fp16", batch=33, head_q=32, head_k=1, dim=256,
             prefix=8192, own=128, page=64, alibi=False, padded=0),
        # a decode step's new rows into a 16-bit cache: one row per sequence, the smallest call
        dict(name="append_decode_16bit", op="append", dtype="bf16", fmt="16", batch=64, head_k=8, dim=128, latent=False,
             old=60, new=1, page=16, fused=True),
        # the same into an int4 cache with a (scale, zero) pair per row
        dict(name="append_decode_int4", op="append", dtype="bf16", fmt="int4_tok", batch=256, head_k=8, dim=128,
             latent=False, old=700, new=1, page=16, fused=True),
        # prompts of many lengths into an int8 cache with a pair per 64 elements
        dict(name="append_prompt_int8", op="append", dtype="fp16", fmt="int8_g64", batch=37, head_k=8, dim=128,
             latent=False, old=300, new=1500, page=64, fused=False),
        # a chunk of prompts into an FP8 latent cache (V inside the K rows)
        dict(name="append_latent_fp8", op="append", dtype="bf16", fmt="fp8", batch=16, head_k=1, dim=576, latent=True,
             old=2000, new=2048, page=64, fused=False),
        # one short conversation read back for a prompt's continuation
        dict(name="read_small", op="read", dtype="bf16", fmt="int8", batch=2, head_k=8, dim=96, latent=False, old=77,
             page=16),
        # whole conversations out of an int4 cache, the largest read
        dict(name="read_int4_large", op="read", dtype="bf16", fmt="int4_g64", batch=64, head_k=8, dim=128, latent=False,
             old=4096, page=16),
        # a 16-bit cache gathered out of its pages
        dict(name="read_16bit", op="read", dtype="fp16", fmt="16", batch=24, head_k=4, dim=256, latent=False, old=1300,
             page=32),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["shared_prefix", "shared_prefix", "append", "append", "read"])
    dtype = rng.choice(["bf16", "fp16"])
    page = rng.choice([1, 16, 32, 64, 256])
    if op == "shared_prefix":
        dim = rng.choice([64, 96, 128, 256])
        head_k = rng.choice([1, 2, 4, 5, 8, 32])
        head_q = head_k * rng.choice([1, 2, 4, 7, 8] if head_k > 2 else [1, 4, 8, 16, 32])
        batch, prefix, most = _log_int(rng, 2, 256), _log_int(rng, 1, 16384), _log_int(rng, 1, 1024)
        while batch * head_q * (prefix + most) > 1 << 26 or batch * most * head_k * dim > 1 << 28:
            prefix, most, batch = (prefix + 1) // 2, (most + 1) // 2, max(2, batch // 2)
        page = rng.choice([0, page])
        if page:
            prefix = max(1, prefix // page) * page
        return dict(op=op, dtype=dtype, batch=batch, head_q=head_q, head_k=head_k, dim=dim, prefix=prefix, own=most,
                    page=page, alibi=rng.random() < 0.3, padded=rng.choice([0, 1]) if page else 0)
    fmt = rng.choice(["16", "fp8", "int8", "int4", "int8_tok", "int4_tok", "int8_g64", "int4_g64"])
    latent = fmt in ("16", "fp8", "int8", "int4") and rng.random() < 0.2
    dim = 576 if latent else rng.choice([64, 128, 256] if "_" in fmt else [64, 96, 128, 256])
    head_k = 1 if latent else rng.choice([1, 2, 4, 5, 8, 32])
    batch, old, new = _log_int(rng, 1, 256), _log_int(rng, 1, 4096), _log_int(rng, 1, 2048)
    if rng.random() < 0.3:
        new = 1
    while batch * (old + new) * head_k * dim > 1 << 28:
        old, new, batch = (old + 1) // 2, (new + 1) // 2, max(1, batch // 2)
    case = dict(op=op, dtype=dtype, fmt=fmt, batch=batch, head_k=head_k, dim=dim, latent=latent, old=old, page=page)
    if op == "append":
        case.update(new=new, fused=rng.random() < 0.5 and not latent)
    return case


def _lengths(bounds, n, g):
    """One column of `n` lengths for each (least, most); the first row holds the most.  Every seed has the same rows, each
    in an order of its own, so that the outputs' sizes are the case's."""
    fixed = torch.Generator().manual_seed(n)
    rows = torch.stack([torch.randint(lo, hi + 1, (n,), generator=fixed, dtype=torch.int64) for lo, hi in bounds], dim=1)
    rows[0] = torch.tensor([hi for _, hi in bounds])
    return rows[torch.randperm(n, generator=g)].unbind(1)


def _cu(lens):
    return torch.nn.functional.pad(lens.cumsum(0), (1, 0)).to(torch.int32)


def _heads(shape, g, dtype):
    """K or V rows: normal, with a spread of magnitudes over the channels."""
    channel = torch.exp(0.5 * torch.randn(shape[-2:], generator=g, device="cuda"))
    return (torch.randn(shape, generator=g, device="cuda") * channel).to(dtype)


def _pages_for(lens, page, extra, g):
    """A block table over shuffled pages for sequences of these lengths, and the number of pages."""
    blocks = (lens + page - 1) // page
    n = int(blocks.sum()) + extra
    order = torch.randperm(n, generator=g)
    width = max(1, int(blocks.max()))
    at = torch.nn.functional.pad(blocks.cumsum(0), (1, 0))[:-1, None] + torch.arange(width)[None, :]
    at = torch.where(torch.arange(width)[None, :] < blocks[:, None], at, torch.zeros_like(at))
    return order[at].to(torch.int32), n, order


def prepare(case, seed):
    gc = torch.Generator().manual_seed(seed)
    g = torch.Generator("cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    if case["op"] == "shared_prefix":
        batch, head_k, dim, prefix = case["batch"], case["head_k"], case["dim"], case["prefix"]
        s = dict(case=case, q=torch.randn(batch, case["head_q"], dim, generator=g, device="cuda").to(dtype))
        own_lens, = _lengths([(0, case["own"])], batch, gc)
        if not case["page"]:
            total = int(own_lens.sum())
            s.update(kp=_heads((prefix, head_k, dim), g, dtype), vp=_heads((prefix, head_k, dim), g, dtype),
                     k=_heads((total, head_k, dim), g, dtype), v=_heads((total, head_k, dim), g, dtype),
                     cu=_cu(own_lens).cuda(), own_max=case["own"])
            return s
        page = case["page"]
        pre_blocks = prefix // page
        table, n, order = _pages_for(own_lens, page, pre_blocks, gc)
        blocks = order[n - pre_blocks:].to(torch.int32)
        lens = own_lens + prefix
        for i in range(min(case["padded"], batch - 1)):  # rows of the batch without a sequence
            lens[batch - 1 - i] = 0
        table = torch.cat([blocks[None, :].expand(batch, -1), table], dim=1).contiguous()
        s.update(k_pages=_heads((n, page, head_k, dim), g, dtype), v_pages=_heads((n, page, head_k, dim), g, dtype),
                 blocks=blocks.cuda(), table=table.cuda(), lens=lens.to(torch.int32).cuda(),
                 max_seq=prefix + case["own"], total=int(lens.sum()), own_max=case["own"])
        return s
    batch, head_k, dim, page, fmt = case["batch"], case["head_k"], case["dim"], case["page"], case["fmt"]
    append = case["op"] == "append"
    if append:
        lens, new = _lengths([(1, case["old"]), (1, case["new"])], batch, gc)
        lens = lens + new
    else:
        lens, = _lengths([(1, case["old"])], batch, gc)
        new = lens
    tokens = int(new.sum())
    table, n, _ = _pages_for(lens, page, 1, gc)
    s = dict(case=case, table=table.cuda(), lens=lens.to(torch.int32).cuda(), tokens=tokens,
             cu=None if append and case["new"] == 1 else _cu(new).cuda())
    kind = fmt.split("_")[0]
    width = dim // 2 if kind == "int4" else dim
    s["k_scale"] = s["v_scale"] = None
    pools = []
    for name in ("k",) if case["latent"] else ("k", "v"):
        if append:
            pool = torch.zeros((n, page, head_k, width), device="cuda", dtype=dtype if kind == "16" else torch.uint8)
        elif kind == "16":
            pool = _heads((n, page, head_k, dim), g, dtype)
        elif kind == "fp8":
            pool = torch.randn((n, page, head_k, dim), generator=g, device="cuda").mul_(60).clamp_(-448, 448)
            pool = pool.to(torch.float8_e4m3fn)
        else:
            pool = torch.randint(0, 256, (n, page, head_k, width), generator=g, device="cuda", dtype=torch.uint8)
        if kind == "fp8":
            pool = pool.view(torch.float8_e4m3fn)
        elif kind == "int8":
            pool = pool.view(torch.int8)
        pools.append(pool)
        if kind == "16":
            continue
        if "_" not in fmt:  # factors that clip a few of the largest values
            at = {"fp8": 448.0, "int8": 127.0, "int4": 7.0}[kind]
            s[name + "_scale"] = 6.0 / at * torch.exp(0.3 * torch.randn(head_k, generator=g, device="cuda"))
        else:
            runs = [n, page, head_k] + ([dim // 64] if fmt.endswith("g64") else [])
            scale = 0.02 * torch.exp(0.3 * torch.randn(runs, generator=g, device="cuda"))
            zero = 3.0 * torch.randn(runs, generator=g, device="cuda")
            pair = torch.stack([scale, zero], dim=-1)
            s[name + "_scale"] = torch.zeros_like(pair) if append else pair
    s["k_pages"], s["v_pages"] = pools[0], None if case["latent"] else pools[1]
    if append:
        if case["fused"]:  # the K and V columns of a fused projection's output
            qkv = _heads((tokens, 3 * head_k, dim), g, dtype)
            s["k"], s["v"] = qkv[:, head_k:2 * head_k], qkv[:, 2 * head_k:]
        else:
            s["k"] = _heads((tokens, head_k, dim), g, dtype)
            s["v"] = None if case["latent"] else _heads((tokens, head_k, dim), g, dtype)
    return s


def _run_own(s):
    import decoding_attention_amd as da
    case = s["case"]
    if case["op"] == "shared_prefix":
        if case["page"]:
            return da.decoding_attn_paged_shared_prefix_fwd(
                s["q"], s["k_pages"], s["v_pages"], s["blocks"], case["prefix"], s["table"], s["lens"], s["max_seq"],
                case["dim"], case["alibi"], total_k=s["total"])
        return da.decoding_attn_shared_prefix_fwd(s["q"], s["kp"], s["vp"], s["k"], s["v"], s["cu"], s["own_max"],
                                                  case["dim"], case["alibi"])
    scales = dict(k_scale=s["k_scale"], v_scale=s["v_scale"])
    if case["op"] == "append":
        da.kv_cache_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["cu"], **scales)
        if case["fmt"] == "16":
            return [s["k_pages"]] + ([] if case["latent"] else [s["v_pages"]])
    k, v = da.kv_cache_read(s["k_pages"], s["v_pages"], s["table"], s["lens"], s["cu"], s["tokens"],
                            dtype=_DTYPES[case["dtype"]], **scales)
    return [k] + ([] if v is None else [v])


def run(state):
    if own:
        return _run_own(state)
    return _plain_prefix(state) if state["case"]["op"] == "shared_prefix" else _plain_cache(state)


def _plain_prefix(s):
    case = s["case"]
    q, prefix, most = s["q"].float(), case["prefix"], s["own_max"]
    batch, head_q, dim = q.shape
    head_k = case["head_k"]
    ratio = head_q // head_k
    j = torch.arange(most, device=q.device)
    if case["page"]:
        page = case["page"]
        kp, vp = (t[s["blocks"].long()].reshape(-1, head_k, dim).float() for t in (s["k_pages"], s["v_pages"]))
        lens = s["lens"].long()
        own_lens = (lens - prefix).clamp_min(0)
        pos = prefix + torch.minimum(j[None, :], (own_lens[:, None] - 1).clamp_min(0))
        at = (pos // page).clamp_max(s["table"].shape[1] - 1)
        rows = torch.gather(s["table"].long(), 1, at) * page + pos % page
        k, v = (t.reshape(-1, head_k, dim)[rows].float() for t in (s["k_pages"], s["v_pages"]))
        none = lens == 0
    else:
        kp, vp = s["kp"].float(), s["vp"].float()
        cu = s["cu"].long()
        own_lens = cu[1:] - cu[:-1]
        rows = (cu[:-1, None] + j[None, :]).clamp_max(max(0, s["k"].shape[0] - 1))
        k, v = (t[rows].float() for t in (s["k"], s["v"]))
        none = torch.zeros_like(own_lens, dtype=torch.bool)
    dead = j[None, :] >= own_lens[:, None]  # [batch, most]
    scale = 1.0 / math.sqrt(dim)
    # prefix: the rows of one KV head are the whole batch's; own tokens: each sequence by itself
    qh = q.view(batch, head_k, ratio, dim)
    sp = torch.matmul(qh.permute(1, 0, 2, 3).reshape(head_k, batch * ratio, dim), kp.permute(1, 2, 0)) * scale
    sp = sp.view(head_k, batch, ratio, prefix).permute(1, 0, 2, 3)
    so = torch.matmul(qh, k.permute(0, 2, 3, 1)) * scale  # [batch, head_k, ratio, most]
    if case["alibi"]:
        slope = torch.exp2(-8.0 * torch.arange(1, head_q + 1, device=q.device) / head_q).view(1, head_k, ratio, 1)
        last = (prefix + own_lens - 1).view(batch, 1, 1, 1)
        sp = sp + slope * (torch.arange(prefix, device=q.device) - last)
        so = so + slope * (prefix + j - last)
    so = so.masked_fill(dead[:, None, None, :], -math.inf)
    m = torch.maximum(sp.amax(-1, keepdim=True), so.amax(-1, keepdim=True))
    pp, po = torch.exp(sp - m), torch.exp(so - m)
    den = pp.sum(-1, keepdim=True) + po.sum(-1, keepdim=True)
    op = torch.matmul(pp.permute(1, 0, 2, 3).reshape(head_k, batch * ratio, prefix), vp.permute(1, 0, 2))
    op = op.view(head_k, batch, ratio, dim).permute(1, 0, 2, 3)
    v = v.masked_fill(dead[:, :, None, None], 0.0)
    o = (op + torch.matmul(po, v.permute(0, 2, 1, 3))) / den
    o = o.masked_fill(none.view(batch, 1, 1, 1), 0.0)
    return o.reshape(batch, head_q, dim).to(s["q"].dtype)


def _rows_of(s):
    """The pools' row of each token: the tokens of a sequence are its last ones."""
    page, lens = s["case"]["page"], s["lens"].long()
    t = torch.arange(s["tokens"], device=lens.device)
    if s["cu"] is None:
        b, pos = t, lens - 1
    else:
        cu = s["cu"].long()
        b = torch.searchsorted(cu, t, right=True) - 1
        pos = lens[b] - (cu[b + 1] - t)
    return s["table"].long()[b, pos // page] * page + pos % page


def _to_e4m3(x):
    """The nearest e4m3 number (ties to even), saturating."""
    x = x.clamp(-448.0, 448.0)
    _, e = torch.frexp(x)
    step = torch.exp2((e - 1).clamp_min(-6).double() - 3.0)
    return torch.round(x / step) * step


def _plain_quantise(x, scale, fmt):
    """(rows as the pool holds them, the (scale, zero) pairs or None) of x [tokens, heads, dim]."""
    kind = fmt.split("_")[0]
    xd = x.double()
    if "_" not in fmt:
        y = xd / scale.double()[None, :, None]
        if kind == "fp8":
            return _to_e4m3(y).float().to(torch.float8_e4m3fn), None
        n, pair = torch.round(y).clamp(_QMIN[kind], _QMAX[kind]), None
    else:
        xr = xd.unflatten(-1, (-1, 64)) if fmt.endswith("g64") else xd[..., None, :]
        lo, hi = xr.amin(-1, keepdim=True), xr.amax(-1, keepdim=True)
        steps = torch.full_like(lo, _QMAX[kind] - _QMIN[kind])
        sc = ((hi - lo) / steps).float().clamp_min(1e-8)
        zero = (_QMIN[kind] - lo / sc.double()).float()
        n = torch.round(xr / sc.double() + zero.double()).clamp(_QMIN[kind], _QMAX[kind]).flatten(-2)
        pair = torch.cat([sc, zero], dim=-1)
        pair = pair if fmt.endswith("g64") else pair[..., 0, :]
    n = n.to(torch.int16)
    if kind == "int8":
        return n.to(torch.int8), pair
    n = n & 15
    return (n[..., 0::2] | (n[..., 1::2] << 4)).to(torch.uint8), pair


def _plain_values(rows, scale, fmt, at):
    """float32 values of pool rows [tokens, heads, width] that lie at rows `at` of the pool."""
    kind = fmt.split("_")[0]
    if kind == "int4":
        r = rows.to(torch.int16)
        n = torch.stack([((r & 15) ^ 8) - 8, ((r >> 4) ^ 8) - 8], dim=-1).flatten(-2).float()
    else:
        n = rows.float()
    if kind == "16":
        return n
    if "_" not in fmt:
        return n * scale[None, :, None]
    pair = scale.flatten(0, 1)[at]
    if fmt.endswith("g64"):
        return (pair[..., :1] * (n.unflatten(-1, (-1, 64)) - pair[..., 1:])).flatten(-2)
    return pair[..., :1] * (n - pair[..., 1:])


def _plain_cache_of(s, name, at):
    case, pool, scale = s["case"], s[name + "_pages"], s[name + "_scale"]
    flat = pool.flatten(0, 1)
    if case["op"] == "append":
        if case["fmt"] == "16":
            flat[at] = s[name]
            return pool
        rows, pair = _plain_quantise(s[name], scale, case["fmt"])
        flat.view(torch.uint8)[at] = rows.view(torch.uint8)
        if pair is not None:
            scale.flatten(0, 1)[at] = pair
    rows = flat.view(torch.uint8)[at].view(flat.dtype) if flat.dtype == torch.float8_e4m3fn else flat[at]
    return _plain_values(rows, scale, case["fmt"], at).to(_DTYPES[case["dtype"]])


def _plain_cache(s):
    at = _rows_of(s)
    return [_plain_cache_of(s, "k", at)] + ([] if s["v_pages"] is None else [_plain_cache_of(s, "v", at)])


def work(case):
    """The bytes and operations of one pass, from the mean lengths of `prepare`'s draws."""
    if case["op"] == "shared_prefix":
        live = case["batch"] - (min(case["padded"], case["batch"] - 1) if case["page"] else 0)
        own_tokens = live * case["own"] / 2
        row = 2 * 2 * case["head_k"] * case["dim"]  # a token's K and V
        rows = (case["prefix"] + own_tokens) * row + 2 * 2 * case["batch"] * case["head_q"] * case["dim"]
        return {"bytes": rows, "flops": 4 * case["head_q"] * case["dim"] * (live * case["prefix"] + own_tokens)}
    fmt = case["fmt"]
    kind = fmt.split("_")[0]
    parts = 1 if case["latent"] else 2
    per = {"16": 2.0, "fp8": 1.0, "int8": 1.0, "int4": 0.5}[kind]
    pairs = 8.0 * (case["dim"] / 64 if fmt.endswith("g64") else 1) if "_" in fmt else 0.0
    held = case["head_k"] * (case["dim"] * per + pairs)
    wide = case["head_k"] * case["dim"] * 2.0
    if case["op"] == "read":
        tokens = case["batch"] * (case["old"] + 1) / 2
        return {"bytes": tokens * parts * (held + wide), "flops": tokens * parts * case["head_k"] * case["dim"] * 2}
    tokens = case["batch"] * (case["new"] + 1) / 2
    # read the new rows, write them; a quantised cache is read back as well
    total = wide + held + (0 if kind == "16" else held + wide)
    return {"bytes": tokens * parts * total, "flops": tokens * parts * case["head_k"] * case["dim"] * 4}


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_prefix(s) if case["op"] == "shared_prefix" else _exact_cache(s)


def _exact_prefix(s):
    case = s["case"]
    q = s["q"].double()
    batch, head_q, dim = q.shape
    prefix, head_k = case["prefix"], case["head_k"]
    ratio = head_q // head_k
    o = torch.zeros_like(q)
    if case["page"]:
        kc, vc = s["k_pages"].flatten(0, 1), s["v_pages"].flatten(0, 1)
        r = torch.arange(prefix, device="cuda")
        pre = s["blocks"].long()[r // case["page"]] * case["page"] + r % case["page"]
        kp, vp = kc[pre], vc[pre]
    else:
        kc, vc, kp, vp = s["k"], s["v"], s["kp"], s["vp"]
    lens = s["lens"].tolist() if case["page"] else None
    cu = None if case["page"] else s["cu"].tolist()
    for h in range(head_k):
        kph, vph = kp[:, h].double(), vp[:, h].double()
        for b in range(batch):
            if case["page"]:
                if lens[b] == 0:
                    continue
                r = torch.arange(prefix, lens[b], device="cuda")
                rows = s["table"][b].long()[r // case["page"]] * case["page"] + r % case["page"]
            else:
                rows = torch.arange(cu[b], cu[b + 1], device="cuda")
            kk = torch.cat([kph, kc[rows, h].double()])
            vv = torch.cat([vph, vc[rows, h].double()])
            heads = slice(h * ratio, (h + 1) * ratio)
            x = q[b, heads] @ kk.T / math.sqrt(dim)
            if case["alibi"]:
                slope = 2.0 ** (-8.0 * torch.arange(h * ratio + 1, (h + 1) * ratio + 1, device="cuda").double() / head_q)
                x += slope[:, None] * (torch.arange(len(kk), device="cuda") - (len(kk) - 1)).double()[None, :]
            o[b, heads] = torch.softmax(x, dim=-1) @ vv
    return o


def _exact_cache(s):
    case = s["case"]
    fmt, page, dim = case["fmt"], case["page"], case["dim"]
    kind = fmt.split("_")[0]
    lens = s["lens"].tolist()
    cu = s["cu"].tolist() if s["cu"] is not None else list(range(case["batch"] + 1))
    rows = []
    for b in range(case["batch"]):
        r = torch.arange(lens[b] - (cu[b + 1] - cu[b]), lens[b], device="cuda")
        rows.append(s["table"][b].long()[r // page] * page + r % page)
    rows = torch.cat(rows)
    out = []
    for name in ("k",) if case["latent"] else ("k", "v"):
        pool, scale = s[name + "_pages"], s[name + "_scale"]
        if case["op"] == "append":
            x = s[name].double()
            if kind == "16":
                full = pool.double().flatten(0, 1)
                full[rows] = x
                out.append(full.view(pool.shape))
                continue
            if "_" not in fmt:
                sc = scale.double().view(1, -1, 1)
                y = x / sc
                if kind == "fp8":
                    a = y.abs().clamp_max(448.0)
                    binade = torch.floor(torch.log2(a.clamp_min(2.0 ** -6)))
                    binade = torch.where(2.0 ** binade > a.clamp_min(2.0 ** -6), binade - 1, binade)
                    ulp = 2.0 ** (binade - 3)
                    out.append(sc * torch.sign(y) * ulp * torch.round(a / ulp))
                else:
                    out.append(sc * torch.round(y).clamp(_QMIN[kind], _QMAX[kind]))
                continue
            run_of = 64 if fmt.endswith("g64") else dim
            xr = x.reshape(x.shape[0], x.shape[1], dim // run_of, run_of)
            lo = xr.min(dim=-1, keepdim=True).values
            hi = xr.max(dim=-1, keepdim=True).values
            levels = torch.tensor(_QMAX[kind] - _QMIN[kind], dtype=torch.float64, device="cuda")
            sc = torch.maximum(((hi - lo) / levels).float(), torch.tensor(1e-8, device="cuda")).double()
            zero = (_QMIN[kind] - lo / sc).float().double()
            n = torch.round(xr / sc + zero).clamp(_QMIN[kind], _QMAX[kind])
            out.append((sc * (n - zero)).reshape(x.shape))
            continue
        flat = pool.flatten(0, 1)
        held = (flat.view(torch.uint8)[rows].view(flat.dtype) if kind == "fp8" else flat[rows])
        if kind == "int4":
            n = torch.empty(len(rows), case["head_k"], dim, dtype=torch.float64, device="cuda")
            low, high = (held % 16).double(), (held // 16).double()
            n[..., 0::2] = torch.where(low >= 8, low - 16, low)
            n[..., 1::2] = torch.where(high >= 8, high - 16, high)
        else:
            n = held.double()
        if kind == "16":
            out.append(n)
        elif "_" not in fmt:
            out.append(n * scale.double().view(1, -1, 1))
        else:
            pair = scale.double().flatten(0, 1)[rows]
            if not fmt.endswith("g64"):
                pair = pair[:, :, None, :]
            nr = n.reshape(n.shape[0], n.shape[1], pair.shape[2], -1)
            out.append((pair[..., 0:1] * (nr - pair[..., 1:2])).reshape(n.shape))
    return out
