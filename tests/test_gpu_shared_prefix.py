"""Attention behind a shared prefix (decoding_attn_shared_prefix_fwd and its paged form) against a float64 softmax.

Tolerance, for a row with weights w over N tokens (u = half a step of the type): every probability is rounded to 16 bits on
its way into the second product and the denominator sums the rounded ones, so that the output moves by at most
u sum w |v - o|; the result is rounded once, u |o|; both products, the sums and the exponential are float32: N 2^-24
sum w |v| for the sums over the tokens, and 2^-20 (1 + max |x|) of the same for scores x, their scale and exp2.  fp16: a
probability below 2^-14 of the largest has an absolute error, at most 2^-25 each; results below 2^-14 likewise.
"""
import math

import pytest
import torch

from decoding_attention_amd import (decoding_attn_fwd, decoding_attn_paged_fwd, decoding_attn_paged_shared_prefix_fwd,
                                    decoding_attn_shared_prefix_fwd, kv_cache_append, kv_cache_read)

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def reference(q, kp, vp, ks, vs, is_alibi, scale=None, slopes=None, live=None):
    """(o, tolerance) in float64: q [batch, heads, dim]; kp, vp the prefix; ks, vs a list of every sequence's own rows."""
    batch, hq, d = q.shape
    hk = kp.shape[1]
    ratio = hq // hk
    u = torch.finfo(q.dtype).eps / 2
    scale = 1 / math.sqrt(d) if scale is None else scale
    o, tol = torch.zeros(batch, hq, d, dtype=torch.float64), torch.zeros(batch, hq, d, dtype=torch.float64)
    for b in range(batch):
        if live is not None and not live[b]:
            continue
        k = torch.cat([kp, ks[b]]).double().repeat_interleave(ratio, dim=1)
        v = torch.cat([vp, vs[b]]).double().repeat_interleave(ratio, dim=1)
        n = k.shape[0]
        if n == 0:
            continue
        x = torch.bmm(k.permute(1, 0, 2).contiguous(), q[b].double()[:, :, None])[..., 0] * scale  # [heads, n]
        if is_alibi:
            s = slopes.double() if slopes is not None else 2.0 ** (-8.0 * torch.arange(1, hq + 1, dtype=torch.float64) / hq)
            x = x + s[:, None] * (torch.arange(n, dtype=torch.float64) - (n - 1))
        w = torch.softmax(x, dim=-1)
        vt = v.permute(1, 0, 2).contiguous()
        o[b] = torch.bmm(w[:, None, :], vt)[:, 0]
        spread = torch.bmm(w[:, None, :], (vt - o[b][:, None, :]).abs())[:, 0]
        size = torch.bmm(w[:, None, :], vt.abs())[:, 0]
        top = x.abs().amax(dim=-1, keepdim=True)
        tol[b] = 1.01 * u * (spread + o[b].abs()) + (n * 2.0 ** -24 + 2.0 ** -20 * (1 + top)) * size
        if q.dtype == torch.float16:
            tol[b] += n * 2.0 ** -25 * vt.abs().amax() + 2.0 ** -25
    return o, tol


def make(batch, hq, hk, d, prefix, own, dtype, seed=0, sharp=1.0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype)  # noqa: E731
    q = (torch.randn(batch, hq, d, generator=g) * sharp).to(dtype)
    kp, vp = r(prefix, hk, d), r(prefix, hk, d)
    ks, vs = [r(n, hk, d) for n in own], [r(n, hk, d) for n in own]
    return q, kp, vp, ks, vs


def packed(ks, vs, hk, d, dtype):
    cu = torch.tensor([0] + [k.shape[0] for k in ks]).cumsum(0).to(torch.int32)
    return torch.cat(ks).to(DEV), torch.cat(vs).to(DEV), cu.to(DEV), max(k.shape[0] for k in ks)


def paged(kp, vp, ks, vs, page, seed=0, padded=()):
    """Pools with shuffled pages, NaN wherever no token lies; the rows' own entries of the prefix are no pages at all."""
    g = torch.Generator().manual_seed(seed)
    pre = kp.shape[0] // page
    assert pre * page == kp.shape[0]
    blocks = [(k.shape[0] + page - 1) // page for k in ks]
    n = pre + sum(blocks) + 2
    order = torch.randperm(n, generator=g).tolist()
    pk = torch.full((n, page) + kp.shape[1:], float("nan"), dtype=kp.dtype)
    pv = pk.clone()
    ids = [order.pop() for _ in range(pre)]
    for i, p in enumerate(ids):
        pk[p], pv[p] = kp[i * page:(i + 1) * page], vp[i * page:(i + 1) * page]
    table = torch.full((len(ks), pre + max(1, max(blocks))), -1, dtype=torch.int32)
    lens = []
    for b, k in enumerate(ks):
        for i in range(blocks[b]):
            p = order.pop()
            table[b, pre + i] = p
            rows = k[i * page:(i + 1) * page]
            pk[p, :rows.shape[0]], pv[p, :rows.shape[0]] = rows, vs[b][i * page:(i + 1) * page]
        lens.append(0 if b in padded else kp.shape[0] + k.shape[0])
    return (pk.to(DEV), pv.to(DEV), torch.tensor(ids, dtype=torch.int32, device=DEV), table.to(DEV),
            torch.tensor(lens, dtype=torch.int32, device=DEV), max(lens))


def check(got, ref):
    o, tol = ref
    got = got.cpu().double()
    assert torch.isfinite(got).all()
    over = ((got - o).abs() - tol).max().item()
    assert over <= 0, f"{over:.3e} over the tolerance; largest error {(got - o).abs().max().item():.3e}"


OWN = [0, 1, 5, 33, 64, 200, 31, 2]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("hq,hk", [(8, 8), (16, 4), (6, 2), (20, 1), (7, 7), (33, 1), (15, 5)])
def test_head_layouts(hq, hk, d, dtype):
    q, kp, vp, ks, vs = make(8, hq, hk, d, 133, OWN, dtype, seed=d + hq)
    k, v, cu, most = packed(ks, vs, hk, d, dtype)
    o = decoding_attn_shared_prefix_fwd(q.to(DEV), kp.to(DEV), vp.to(DEV), k, v, cu, most, d, False)
    check(o, reference(q, kp, vp, ks, vs, False))


@pytest.mark.parametrize("prefix", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 1000, 4097])
@pytest.mark.parametrize("d", [64, 96, 128, 256])
def test_prefix_lengths(prefix, d):
    dtype = torch.bfloat16 if prefix % 2 else torch.float16
    q, kp, vp, ks, vs = make(3, 8, 4, d, prefix, [0, 7, 130], dtype, seed=prefix)
    k, v, cu, most = packed(ks, vs, 4, d, dtype)
    o = decoding_attn_shared_prefix_fwd(q.to(DEV), kp.to(DEV), vp.to(DEV), k, v, cu, most, d, False)
    check(o, reference(q, kp, vp, ks, vs, False))


@pytest.mark.parametrize("batch", [1, 2, 31, 32, 33, 65, 130])
@pytest.mark.parametrize("d", [64, 128])
def test_batch_sizes(batch, d):
    """Row tiles that end inside a wave, a work-group, and several of them."""
    own = [(b * 37) % 50 for b in range(batch)]
    q, kp, vp, ks, vs = make(batch, 8, 2, d, 300, own, torch.bfloat16, seed=batch)
    k, v, cu, most = packed(ks, vs, 2, d, torch.bfloat16)
    o = decoding_attn_shared_prefix_fwd(q.to(DEV), kp.to(DEV), vp.to(DEV), k, v, cu, most, d, False)
    check(o, reference(q, kp, vp, ks, vs, False))


@pytest.mark.parametrize("custom", [False, True])
@pytest.mark.parametrize("d,hq,hk", [(64, 8, 8), (128, 16, 4), (256, 20, 1), (96, 12, 3)])
def test_alibi_and_scale(d, hq, hk, custom):
    q, kp, vp, ks, vs = make(8, hq, hk, d, 517, OWN, torch.float16, seed=d)
    k, v, cu, most = packed(ks, vs, hk, d, torch.float16)
    scale, slopes = (0.031, torch.rand(hq) * 0.1) if custom else (None, None)
    o = decoding_attn_shared_prefix_fwd(q.to(DEV), kp.to(DEV), vp.to(DEV), k, v, cu, most, d, True, softmax_scale=scale,
                                        alibi_slopes=None if slopes is None else slopes.to(DEV))
    check(o, reference(q, kp, vp, ks, vs, True, scale, slopes))


@pytest.mark.parametrize("page", [0, 4, 16, 64])
@pytest.mark.parametrize("d", [64, 96, 128, 256])
def test_alibi_over_many_tiles(d, page):
    """Splits of many tiles and a last one that is cut; flat, steep and falling slopes."""
    heads, batch = 64, 3
    prefix = {0: 3003, 4: 3004, 16: 2992, 64: 2944}[page]
    q, kp, vp, ks, vs = make(batch, heads, heads, d, prefix, [0, 3, 40], torch.float16 if d == 64 else torch.bfloat16, seed=d + page)
    slopes = torch.linspace(-0.02, 0.8, heads)
    if page:
        pk, pv, ids, table, lens, most = paged(kp, vp, ks, vs, page, seed=page)
        o = decoding_attn_paged_shared_prefix_fwd(q.to(DEV), pk, pv, ids, prefix, table, lens, most, d, True, alibi_slopes=slopes.to(DEV))
    else:
        k, v, cu, most = packed(ks, vs, heads, d, q.dtype)
        o = decoding_attn_shared_prefix_fwd(q.to(DEV), kp.to(DEV), vp.to(DEV), k, v, cu, most, d, True, alibi_slopes=slopes.to(DEV))
    check(o, reference(q, kp, vp, ks, vs, True, None, slopes))


@pytest.mark.parametrize("page", [1, 2, 8, 16, 32, 64, 256])
@pytest.mark.parametrize("d,hq,hk,alibi", [(128, 16, 4, False), (64, 6, 2, True), (96, 8, 8, False), (256, 33, 1, True)])
def test_pages(d, hq, hk, alibi, page):
    """Own tokens that end inside pages, rows of the batch without a sequence, poisoned unused rows."""
    prefix = 256 if page == 256 else 192
    q, kp, vp, ks, vs = make(8, hq, hk, d, prefix, OWN, torch.bfloat16, seed=page + d)
    pk, pv, ids, table, lens, most = paged(kp, vp, ks, vs, page, seed=page, padded=(2, 7))
    o = decoding_attn_paged_shared_prefix_fwd(q.to(DEV), pk, pv, ids, prefix, table, lens, most, d, alibi)
    check(o, reference(q, kp, vp, ks, vs, alibi, live=[b not in (2, 7) for b in range(8)]))
    assert (o[2] == 0).all() and (o[7] == 0).all()


def test_sequences_shorter_than_the_prefix_get_zero_rows():
    q, kp, vp, ks, vs = make(4, 8, 4, 128, 64, [10, 0, 3, 0], torch.float16)
    pk, pv, ids, table, lens, most = paged(kp, vp, ks, vs, 16)
    lens[3] = 63
    o = decoding_attn_paged_shared_prefix_fwd(q.to(DEV), pk, pv, ids, 64, table, lens, most, 128, False)
    check(o, reference(q, kp, vp, ks, vs, False, live=[True, True, True, False]))


def test_combined_pool_views():
    q, kp, vp, ks, vs = make(4, 8, 4, 128, 64, [10, 40, 3, 0], torch.float16)
    pk, pv, ids, table, lens, most = paged(kp, vp, ks, vs, 16)
    pool = torch.stack([pk, pv], dim=1).contiguous()
    o = decoding_attn_paged_shared_prefix_fwd(q.to(DEV), pool[:, 0], pool[:, 1], ids, 64, table, lens, most, 128, False)
    check(o, reference(q, kp, vp, ks, vs, False))


def test_no_prefix_and_no_own_tokens():
    q, kp, vp, ks, vs = make(4, 8, 4, 128, 100, [0, 0, 0, 0], torch.bfloat16)
    k, v, cu, most = packed(ks, vs, 4, 128, torch.bfloat16)
    args = q.to(DEV), kp.to(DEV), vp.to(DEV)
    check(decoding_attn_shared_prefix_fwd(*args, k, v, cu, most, 128, False), reference(q, kp, vp, ks, vs, False))
    # (a bound that no sequence reaches)
    check(decoding_attn_shared_prefix_fwd(*args, k, v, cu, 500, 128, False), reference(q, kp, vp, ks, vs, False))
    none = kp[:0].to(DEV)
    assert (decoding_attn_shared_prefix_fwd(q.to(DEV), none, none, k, v, cu, most, 128, False) == 0).all()
    q, kp, vp, ks, vs = make(4, 8, 4, 128, 0, [3, 0, 70, 9], torch.bfloat16)
    k, v, cu, most = packed(ks, vs, 4, 128, torch.bfloat16)
    o = decoding_attn_shared_prefix_fwd(q.to(DEV), none, none, k, v, cu, most, 128, False)
    assert torch.equal(o, decoding_attn_fwd(q.to(DEV), k, v, cu, most, 128, False))
    pk, pv, ids, table, lens, most = paged(kp, vp, ks, vs, 16)
    o = decoding_attn_paged_shared_prefix_fwd(q.to(DEV), pk, pv, ids, 0, table, lens, most, 128, False)
    assert torch.equal(o, decoding_attn_paged_fwd(q.to(DEV), pk, pv, table, lens, most, 128, False))


@pytest.mark.parametrize("sharp", [0.0, 8.0, 60.0])
def test_flat_and_steep_scores(sharp):
    """Equal weights, and one token that takes all the weight, in the prefix or behind it."""
    q, kp, vp, ks, vs = make(8, 8, 2, 128, 700, OWN, torch.bfloat16, seed=4, sharp=sharp)
    k, v, cu, most = packed(ks, vs, 2, 128, torch.bfloat16)
    o = decoding_attn_shared_prefix_fwd(q.to(DEV), kp.to(DEV), vp.to(DEV), k, v, cu, most, 128, False)
    check(o, reference(q, kp, vp, ks, vs, False))


@pytest.mark.parametrize("d", [64, 96, 128, 256])
def test_a_maximum_that_rises_all_the_way(d):
    """Keys in the order of their scores: the running maximum is raised again and again."""
    q, kp, vp, ks, vs = make(4, 4, 1, d, 2000, [3, 300, 0, 9], torch.float16, seed=5, sharp=0.1)
    ramp = torch.linspace(-60, 60, 2000)
    q[:, :, 0], kp[:, 0, 0] = 8.0, ramp.half()
    k, v, cu, most = packed(ks, vs, 1, d, torch.float16)
    o = decoding_attn_shared_prefix_fwd(q.to(DEV), kp.to(DEV), vp.to(DEV), k, v, cu, most, d, False)
    check(o, reference(q, kp, vp, ks, vs, False))


def test_non_finite_values_stay_with_their_sequences():
    """A NaN among one sequence's own tokens reaches that sequence alone; one in the prefix reaches all."""
    q, kp, vp, ks, vs = make(6, 8, 4, 128, 128, [4, 50, 0, 9, 33, 1], torch.bfloat16, seed=6)
    vs[1][7, 2, 5] = float("nan")
    ks[4][0, 0, 0] = float("inf")
    k, v, cu, most = packed(ks, vs, 4, 128, torch.bfloat16)
    o = decoding_attn_shared_prefix_fwd(q.to(DEV), kp.to(DEV), vp.to(DEV), k, v, cu, most, 128, False).cpu()
    assert torch.isnan(o[1, 4:6, 5]).all() and torch.isfinite(o[[0, 2, 3, 5]]).all()
    kp[100, 1] = float("nan")
    o = decoding_attn_shared_prefix_fwd(q.to(DEV), kp.to(DEV), vp.to(DEV), k, v, cu, most, 128, False).cpu()
    assert torch.isnan(o[:, 2:4]).all() and torch.isfinite(o[[0, 2, 3, 5]][:, :2]).all()


def test_long_prefix_and_large_batch():
    """Many splits, several row tiles, a prefix beyond one split of each; spot checks."""
    own = [(b * 53) % 700 for b in range(200)]
    q, kp, vp, ks, vs = make(200, 32, 8, 128, 9001, own, torch.bfloat16, seed=7)
    k, v, cu, most = packed(ks, vs, 8, 128, torch.bfloat16)
    o = decoding_attn_shared_prefix_fwd(q.to(DEV), kp.to(DEV), vp.to(DEV), k, v, cu, most, 128, False)
    rows = [0, 31, 32, 63, 64, 99, 128, 199]
    check(o[rows], reference(q[rows], kp, vp, [ks[b] for b in rows], [vs[b] for b in rows], False))


def test_same_bits_twice_and_on_another_stream():
    q, kp, vp, ks, vs = make(8, 16, 4, 128, 900, OWN, torch.bfloat16, seed=8)
    k, v, cu, most = packed(ks, vs, 4, 128, torch.bfloat16)
    args = (q.to(DEV), kp.to(DEV), vp.to(DEV), k, v, cu, most, 128, False)
    a = decoding_attn_shared_prefix_fwd(*args)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = decoding_attn_shared_prefix_fwd(*args)
    c = decoding_attn_shared_prefix_fwd(*args)  # (both streams at once)
    torch.cuda.synchronize()
    assert torch.equal(a, b) and torch.equal(a, c)


def test_replays_from_a_graph_with_other_lengths():
    """Two captured graphs of one call, replayed with eager work between; the lengths live on the device."""
    q, kp, vp, ks, vs = make(8, 16, 4, 128, 256, OWN, torch.bfloat16, seed=9)
    pk, pv, ids, table, lens, most = paged(kp, vp, ks, vs, 16)
    dq = q.to(DEV)

    def run():
        return decoding_attn_paged_shared_prefix_fwd(dq, pk, pv, ids, 256, table, lens, most, 128, False)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run()
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        graphs.append((graph, out))
    g = torch.Generator().manual_seed(10)
    full = lens.clone()
    for step in range(4):
        dq.copy_(torch.randn(q.shape, generator=g).to(q.dtype))
        lens.copy_(torch.where(torch.arange(8, device=DEV) == step, torch.zeros_like(full), full - (full > 256).int() * step % 2))
        for graph, out in graphs:
            graph.replay()
        want = run()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert torch.equal(out, want)
        assert (want[step] == 0).all()


def test_entry_point_with_its_own_and_the_callers_workspace():
    from decoding_attention_amd import _lib
    lib = _lib.load()
    q, kp, vp, ks, vs = make(8, 16, 4, 128, 300, OWN, torch.float16, seed=11)
    k, v, cu, most = packed(ks, vs, 4, 128, torch.float16)
    dq, dkp, dvp = q.to(DEV), kp.to(DEV), vp.to(DEV)
    need = lib.da_workspace_bytes_shared_prefix(300, most, 8, 16, 4, 128, 128, k.shape[0], 0)
    ws = torch.full((need,), 255, dtype=torch.uint8, device=DEV)  # (NaN everywhere)
    outs = []
    for ptr, size in ((ws.data_ptr(), need), (None, 0)):
        o = torch.full((8, 16, 128), float("nan"), dtype=torch.float16, device=DEV)
        call = lambda b: lib.da_decoding_attn_shared_prefix(  # noqa: E731
            dq.data_ptr(), dkp.data_ptr(), dvp.data_ptr(), 300, k.data_ptr(), v.data_ptr(), o.data_ptr(), cu.data_ptr(), most,
            8, 16, 4, 128, 128, 0, 0, 0.0, None, k.shape[0], ptr, b, torch.cuda.current_stream().cuda_stream)
        assert call(size) == 0, _lib.last_error()
        torch.cuda.synchronize()
        outs.append(o)
        if ptr:
            assert call(size - 16) == _lib.DA_ERR_WORKSPACE
    check(outs[0], reference(q, kp, vp, ks, vs, False))
    assert torch.equal(outs[0], outs[1])
    assert lib.da_release_workspaces() == 0


def test_a_serving_loop():
    """The operators together: a prefix and prompts appended to a paged cache, decode steps that append a row per sequence and
    attend behind the prefix, and the cache read back at the end.  Every step against float64, and against the attention that
    reads the whole block table."""
    hk, hq, d, page, prefix, dtype = 4, 16, 128, 16, 160, torch.bfloat16
    prompts = [17, 1, 40, 0, 64]
    steps, batch = 4, 5
    own = [n + steps for n in prompts]
    q, kp, vp, ks, vs = make(batch, hq, hk, d, prefix, own, dtype, seed=12)
    pk, pv, ids, table, lens, most = paged(kp, vp, ks, vs, page, seed=13)
    pk.fill_(0), pv.fill_(0)
    # the prefix is written once, through the first sequence's pages
    table[:, :prefix // page] = ids
    kv_cache_append(kp.to(DEV), vp.to(DEV), pk, pv, table[:1].contiguous(), torch.tensor([prefix], dtype=torch.int32, device=DEV),
                    torch.tensor([0, prefix], dtype=torch.int32, device=DEV))
    cu = torch.tensor([0] + prompts).cumsum(0).to(torch.int32).to(DEV)
    now = torch.tensor([prefix + n for n in prompts], dtype=torch.int32, device=DEV)
    kv_cache_append(torch.cat([k[:n] for k, n in zip(ks, prompts)]).to(DEV), torch.cat([v[:n] for v, n in zip(vs, prompts)]).to(DEV),
                    pk, pv, table, now, cu)
    g = torch.Generator().manual_seed(14)
    for step in range(steps):
        now += 1
        kv_cache_append(torch.stack([k[n + step] for k, n in zip(ks, prompts)]).to(DEV),
                        torch.stack([v[n + step] for v, n in zip(vs, prompts)]).to(DEV), pk, pv, table, now)
        q = torch.randn(batch, hq, d, generator=g).to(dtype)
        o = decoding_attn_paged_shared_prefix_fwd(q.to(DEV), pk, pv, ids, prefix, table, now, most, d, False)
        seen_k, seen_v = ([t[:n + step + 1] for t, n in zip(x, prompts)] for x in (ks, vs))
        ref = reference(q, kp, vp, seen_k, seen_v, False)
        check(o, ref)
        check(decoding_attn_paged_fwd(q.to(DEV), pk, pv, table, now, most, d, False), ref)
    assert torch.equal(now, lens)
    cu = torch.cat([torch.zeros(1, dtype=torch.int32, device=DEV), lens.cumsum(0).to(torch.int32)])
    k, v = kv_cache_read(pk, pv, table, lens, cu, int(cu[-1]), dtype=dtype)
    assert torch.equal(k.cpu(), torch.cat([torch.cat([kp, t]) for t in ks]))
    assert torch.equal(v.cpu(), torch.cat([torch.cat([vp, t]) for t in vs]))


def some(q, kp, vp, ks, vs, alibi, rows, padded=()):
    """The reference of a few of the batch's rows."""
    return reference(q[rows], kp, vp, [ks[b] for b in rows], [vs[b] for b in rows], alibi, live=[b not in padded for b in rows])


# enough own tokens for equal shares of them, whatever the sequences' lengths: none, one, many shares long
LONG_OWN = [0, 1, 3000, 17, 128, 0, 5000, 31, 32, 33, 900, 0, 64, 2500, 1, 1, 700, 4096, 129, 0]


@pytest.mark.parametrize("page", [0, 1, 4, 8, 16, 32, 128])
@pytest.mark.parametrize("d,hq,hk,alibi", [(128, 32, 8, False), (64, 34, 1, True), (96, 9, 3, False), (256, 36, 2, False), (128, 7, 7, True)])
def test_own_tokens_in_equal_shares(d, hq, hk, alibi, page):
    """Head groups (more than sixteen rows to a KV head), a wave per head and a head per work-group; padded rows."""
    prefix, dtype, rows = 384, torch.float16 if page == 4 else torch.bfloat16, [0, 1, 2, 5, 6, 10, 13, 19]
    q, kp, vp, ks, vs = make(len(LONG_OWN), hq, hk, d, prefix, LONG_OWN, dtype, seed=d + page)
    padded = (5, 10) if page else ()
    if page:
        pk, pv, ids, table, lens, most = paged(kp, vp, ks, vs, page, seed=page, padded=padded)
        o = decoding_attn_paged_shared_prefix_fwd(q.to(DEV), pk, pv, ids, prefix, table, lens, most, d, alibi,
                                                  total_k=int(lens.sum()))
    else:
        k, v, cu, most = packed(ks, vs, hk, d, dtype)
        o = decoding_attn_shared_prefix_fwd(q.to(DEV), kp.to(DEV), vp.to(DEV), k, v, cu, most, d, alibi)
    assert torch.isfinite(o).all()
    check(o[rows], some(q, kp, vp, ks, vs, alibi, rows, padded))


@pytest.mark.parametrize("batch", [1023, 1024, 1025])
@pytest.mark.parametrize("page", [0, 16])
def test_around_the_largest_batch_of_equal_shares(batch, page):
    own = [(b * 41) % 150 for b in range(batch)]
    own[-1] = 77
    q, kp, vp, ks, vs = make(batch, 4, 4, 64, 64, own, torch.bfloat16, seed=batch)
    rows = [0, 1, 255, 256, 500, 767, 768, 1022, batch - 1]
    if page:
        pk, pv, ids, table, lens, most = paged(kp, vp, ks, vs, page, seed=page, padded=(500,))
        o = decoding_attn_paged_shared_prefix_fwd(q.to(DEV), pk, pv, ids, 64, table, lens, most, 64, False)
    else:
        k, v, cu, most = packed(ks, vs, 4, 64, torch.bfloat16)
        o = decoding_attn_shared_prefix_fwd(q.to(DEV), kp.to(DEV), vp.to(DEV), k, v, cu, most, 64, False)
    assert torch.isfinite(o).all()
    check(o[rows], some(q, kp, vp, ks, vs, False, rows, (500,) if page else ()))


@pytest.mark.parametrize("total_k", [0, 1, 384, 10 ** 9])
def test_hints_move_no_result_out_of_tolerance(total_k):
    """total_k and the bound on the lengths are hints: wrong ones plan badly, and change roundings at most."""
    prefix, rows = 384, [0, 1, 2, 6, 13, 19]
    q, kp, vp, ks, vs = make(len(LONG_OWN), 32, 8, 128, prefix, LONG_OWN, torch.bfloat16, seed=1)
    pk, pv, ids, table, lens, most = paged(kp, vp, ks, vs, 16, seed=1)
    table = torch.nn.functional.pad(table, (0, 300), value=-1)
    for bound in (most, most + 4000):
        o = decoding_attn_paged_shared_prefix_fwd(q.to(DEV), pk, pv, ids, prefix, table, lens, bound, 128, False, total_k=total_k)
        check(o[rows], some(q, kp, vp, ks, vs, False, rows))
    k, v, cu, most = packed(ks, vs, 8, 128, torch.bfloat16)
    o = decoding_attn_shared_prefix_fwd(q.to(DEV), kp.to(DEV), vp.to(DEV), k, v, cu, 3 * most, 128, False)
    check(o[rows], some(q, kp, vp, ks, vs, False, rows))


@pytest.mark.parametrize("page", [0, 1, 16, 64])
def test_replays_of_equal_shares_with_other_lengths(page):
    """The shares follow the lengths on the device: shorter sequences, empty ones, and none at all under the captured plan."""
    prefix, d = 256, 128
    q, kp, vp, ks, vs = make(len(LONG_OWN), 32, 8, d, prefix, LONG_OWN, torch.bfloat16, seed=20 + page)
    dq = q.to(DEV)
    if page:
        pk, pv, ids, table, lens, most = paged(kp, vp, ks, vs, page, seed=page)
        run = lambda: decoding_attn_paged_shared_prefix_fwd(dq, pk, pv, ids, prefix, table, lens, most, d, False)  # noqa: E731
    else:
        k, v, cu, most = packed(ks, vs, 8, d, torch.bfloat16)
        dkp, dvp = kp.to(DEV), vp.to(DEV)
        run = lambda: decoding_attn_shared_prefix_fwd(dq, dkp, dvp, k, v, cu, most, d, False)  # noqa: E731
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run()
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        graphs.append((graph, out))
    g = torch.Generator().manual_seed(21)
    for step in range(4):
        own = [0 if step == 2 else max(0, n - step * 37) for n in LONG_OWN]
        if page:
            lens.copy_(torch.tensor([0 if step == 3 and b % 3 == 0 else prefix + n for b, n in enumerate(own)], dtype=torch.int32))
        else:
            cu.copy_(torch.tensor([0] + own).cumsum(0).to(torch.int32))
        dq.copy_(torch.randn(q.shape, generator=g).to(q.dtype))
        for graph, out in graphs:
            graph.replay()
        want = run()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert torch.equal(out, want)
        if page:  # (the packed rows move with the lengths)
            rows, padded = [0, 1, 2, 6, 13], [b for b in range(20) if step == 3 and b % 3 == 0]
            cut = lambda x: [t[:n] for t, n in zip(x, own)]  # noqa: E731
            check(want[rows], some(dq.cpu(), kp, vp, cut(ks), cut(vs), False, rows, padded))


def test_row_tiles_over_all_chiplets():
    """Two KV heads of 21 row tiles each, few splits: more tiles than one chiplet's share of the pairs would hold."""
    own = [(b * 7) % 9 for b in range(82)]
    q, kp, vp, ks, vs = make(82, 64, 2, 64, 2080, own, torch.float16, seed=22)
    k, v, cu, most = packed(ks, vs, 2, 64, torch.float16)
    o = decoding_attn_shared_prefix_fwd(q.to(DEV), kp.to(DEV), vp.to(DEV), k, v, cu, most, 64, False)
    rows = [0, 3, 4, 40, 41, 80, 81]
    check(o[rows], some(q, kp, vp, ks, vs, False, rows))


@pytest.mark.parametrize("page", [2, 16, 64])
def test_pages_past_32_bit_offsets(page):
    """Prefix and own pages at both ends of pools of more than 2^32 elements."""
    hk, d, prefix, own = 8, 128, 192, [0, 5, 70, 1]
    q, kp, vp, ks, vs = make(4, 32, hk, d, prefix, own, torch.bfloat16, seed=23)
    pk, pv, ids, table, lens, most = paged(kp, vp, ks, vs, page, seed=23)
    n = pk.shape[0]
    pages = 4_400_000_000 // (page * hk * d)
    far = pages - n + torch.arange(n, device=DEV)  # (every second page at the start)
    where = torch.where(torch.arange(n, device=DEV) % 2 == 0, torch.arange(n, device=DEV), far)
    big = [torch.empty(pages, page, hk, d, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    for pool, small in zip(big, (pk, pv)):
        for i, w in enumerate(where.tolist()):
            pool[w].copy_(small[i])
    table = torch.where(table >= 0, where[table.clamp(min=0).long()], -1).to(torch.int32)
    o = decoding_attn_paged_shared_prefix_fwd(q.to(DEV), *big, where[ids.long()].to(torch.int32), prefix, table, lens, most, d, False)
    check(o, reference(q, kp, vp, ks, vs, False))


@pytest.mark.parametrize("lengths", [OWN, LONG_OWN], ids=["short", "long"])
@pytest.mark.parametrize("page", [0, 1, 16, 64])
def test_bounds_below_the_lengths_drop_no_token(page, lengths):
    """A bound on the lengths that is too low, down to the prefix's own length (no own token at all) and to zero: the tokens that
    the device's lengths name are attended to all the same."""
    prefix, hq, hk, d = 192, 16, 4, 128
    q, kp, vp, ks, vs = make(len(lengths), hq, hk, d, prefix, lengths, torch.bfloat16, seed=30 + page)
    rows = [0, 1, 2, 4, 6, 7]
    ref = some(q, kp, vp, ks, vs, False, rows)
    if page:
        pk, pv, ids, table, lens, _ = paged(kp, vp, ks, vs, page, seed=page)
        for bound in (0, 1, prefix, prefix + 1, prefix + 40):
            for total in (0, int(lens.sum())):
                o = decoding_attn_paged_shared_prefix_fwd(q.to(DEV), pk, pv, ids, prefix, table, lens, bound, d, False, total_k=total)
                check(o[rows], ref)
    else:
        k, v, cu, _ = packed(ks, vs, hk, d, torch.bfloat16)
        for bound in (0, 1, 40):
            o = decoding_attn_shared_prefix_fwd(q.to(DEV), kp.to(DEV), vp.to(DEV), k, v, cu, bound, d, False)
            check(o[rows], ref)


def test_entry_point_with_a_bound_of_zero():
    """The C call with rows and max_seq_k 0 attends to them; with max_seq_k 0 and no rows the prefix is all there is.  The
    workspace that the query names for a bound of zero covers both."""
    from decoding_attention_amd import _lib
    lib = _lib.load()
    for prefix in (300, 5000):
        q, kp, vp, ks, vs = make(8, 16, 4, 128, prefix, OWN, torch.float16, seed=31)
        k, v, cu, _ = packed(ks, vs, 4, 128, torch.float16)
        dq, dkp, dvp = q.to(DEV), kp.to(DEV), vp.to(DEV)
        need = lib.da_workspace_bytes_shared_prefix(prefix, 0, 8, 16, 4, 128, 128, 0, 0)
        none = [t[:0] for t in ks]
        for rows in (True, False):
            ws = torch.full((need,), 255, dtype=torch.uint8, device=DEV)
            o = torch.full((8, 16, 128), float("nan"), dtype=torch.float16, device=DEV)
            at = cu if rows else torch.zeros_like(cu)
            rc = lib.da_decoding_attn_shared_prefix(
                dq.data_ptr(), dkp.data_ptr(), dvp.data_ptr(), prefix, k.data_ptr() if rows else None,
                v.data_ptr() if rows else None, o.data_ptr(), at.data_ptr(), 0, 8, 16, 4, 128, 128, 0, 0, 0.0, None, 0,
                ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
            assert rc == 0, _lib.last_error()
            torch.cuda.synchronize()
            check(o, reference(q, kp, vp, ks if rows else none, vs if rows else none, False))


def check_infinite(got, ref, at):
    """As check(), with entries (sequence or slice, heads, column, +-inf) that have to be that infinity."""
    got = got.cpu().clone()
    for b, heads, col, value in at:
        assert (got[b, heads, col] == value).all(), got[b, heads, col]
        got[b, heads, col] = 0
        ref[0][b, heads, col] = 0
    check(got, ref)


@pytest.mark.parametrize("alibi", [False, True])
@pytest.mark.parametrize("prefix,page", [(1, 0), (31, 0), (33, 0), (77, 0), (100, 0), (1001, 0), (5, 1), (100, 4), (1004, 4), (48, 16)])
@pytest.mark.parametrize("d", [64, 96, 128, 256])
def test_an_infinite_value_in_the_prefixs_last_token(d, prefix, page, alibi):
    """Every sequence gives it weight, so that it is infinite in its column of the KV head's rows and nowhere else: what fills up
    the last tile of a prefix that is no multiple of 32 tokens has weight zero, and zero times infinity is no number."""
    hq, hk, dtype = 12, 3, torch.bfloat16 if prefix % 2 else torch.float16
    q, kp, vp, ks, vs = make(5, hq, hk, d, prefix, [0, 3, 40, 1, 0], dtype, seed=prefix + d)
    vp[-1, 1, 3] = vp[-1, 1, d - 1] = 0.0
    slopes = torch.full((hq,), 0.02) if alibi else None
    ref = reference(q, kp, vp, ks, vs, alibi, None, slopes)
    vp[-1, 1, 3], vp[-1, 1, d - 1] = float("inf"), -float("inf")
    dslopes = slopes.to(DEV) if alibi else None
    if page:
        pk, pv, ids, table, lens, most = paged(kp, vp, ks, vs, page, seed=page)
        o = decoding_attn_paged_shared_prefix_fwd(q.to(DEV), pk, pv, ids, prefix, table, lens, most, d, alibi, alibi_slopes=dslopes)
    else:
        k, v, cu, most = packed(ks, vs, hk, d, dtype)
        o = decoding_attn_shared_prefix_fwd(q.to(DEV), kp.to(DEV), vp.to(DEV), k, v, cu, most, d, alibi, alibi_slopes=dslopes)
    check_infinite(o, ref, [(slice(None), slice(4, 8), 3, float("inf")), (slice(None), slice(4, 8), d - 1, -float("inf"))])


@pytest.mark.parametrize("prefix", [1984, 2003])
@pytest.mark.parametrize("falling", [False, True])
@pytest.mark.parametrize("d", [64, 96, 128, 256])
def test_a_maximum_that_moves_in_splits_of_many_tiles(d, falling, prefix):
    """Keys in the order of their scores, up or down, in splits whose last tile is whole or cut: from either end of a split the
    running maximum is raised again and again, and the values far from it still count for nothing."""
    heads = 64
    q, kp, vp, ks, vs = make(3, heads, heads, d, prefix, [0, 3, 40], torch.bfloat16, seed=5 + d, sharp=0.1)
    ramp = torch.linspace(-60, 60, prefix)
    q[:, :, 0], kp[:, :, 0] = 8.0, (ramp.flip(0) if falling else ramp).bfloat16()[:, None]
    k, v, cu, most = packed(ks, vs, heads, d, torch.bfloat16)
    o = decoding_attn_shared_prefix_fwd(q.to(DEV), kp.to(DEV), vp.to(DEV), k, v, cu, most, d, False)
    check(o, reference(q, kp, vp, ks, vs, False))


@pytest.mark.parametrize("lengths", [[0, 3, 40, 32, 1, 133, 16, 47], LONG_OWN], ids=["short", "long"])
@pytest.mark.parametrize("page", [0, 1, 16, 64])
@pytest.mark.parametrize("d,hq,hk", [(64, 4, 4), (96, 12, 3), (128, 16, 4), (256, 33, 1)])
def test_an_infinite_value_in_a_sequences_last_token(d, hq, hk, page, lengths):
    """The same among the own tokens: the sequence's own column, and no other sequence's."""
    prefix, dtype = 64, torch.bfloat16
    q, kp, vp, ks, vs = make(len(lengths), hq, hk, d, prefix, lengths, dtype, seed=page + d)
    rows = [1, 2, 3, 4, 5, 6]
    hit = [b for b in rows if lengths[b] > 0]
    for b in hit:
        vs[b][-1, hk - 1, 5] = 0.0
    ref = some(q, kp, vp, ks, vs, False, rows)
    for b in hit:
        vs[b][-1, hk - 1, 5] = float("inf")
    if page:
        pk, pv, ids, table, lens, most = paged(kp, vp, ks, vs, page, seed=page)
        o = decoding_attn_paged_shared_prefix_fwd(q.to(DEV), pk, pv, ids, prefix, table, lens, most, d, False, total_k=int(lens.sum()))
    else:
        k, v, cu, most = packed(ks, vs, hk, d, dtype)
        o = decoding_attn_shared_prefix_fwd(q.to(DEV), kp.to(DEV), vp.to(DEV), k, v, cu, most, d, False)
    heads = slice((hk - 1) * (hq // hk), hq)
    check_infinite(o[rows], ref, [(rows.index(b), heads, 5, float("inf")) for b in hit])


@pytest.mark.parametrize("page", [0, 16])
@pytest.mark.parametrize("hq,hk", [(1, 1), (3, 1), (4, 4)])
def test_a_hundred_thousand_sequences(hq, hk, page):
    """More sequences than a grid's other axes number, with few rows each; spot checks, and every row is written."""
    batch, d, prefix = 100_003, 64, 48
    own = [(b * 7) % 3 for b in range(batch)]
    g = torch.Generator().manual_seed(hq)
    q = torch.randn(batch, hq, d, generator=g).half()
    kp, vp = (torch.randn(prefix, hk, d, generator=g).half() for _ in range(2))
    cu = torch.tensor([0] + own).cumsum(0)
    k, v = (torch.randn(int(cu[-1]), hk, d, generator=g).half() for _ in range(2))
    rows = [0, 1, 2, 1023, 65535, 65536, 99_999, batch - 1]
    ks, vs = ([t[cu[b]:cu[b + 1]] for b in rows] for t in (k, v))
    if page:
        # a page per sequence behind the prefix's three, its first rows the sequence's own
        pk, pv = (torch.full((3 + batch, page, hk, d), float("nan"), dtype=torch.float16) for _ in range(2))
        seq = torch.repeat_interleave(torch.arange(batch), torch.tensor(own))
        at = torch.arange(len(seq)) - cu[seq]
        for pool, pre, rest in ((pk, kp, k), (pv, vp, v)):
            pool[:3] = pre.unflatten(0, (3, page))
            pool[3 + seq, at] = rest
        ids = torch.arange(3, dtype=torch.int32, device=DEV)
        table = torch.full((batch, 4), -1, dtype=torch.int32)
        table[:, 3] = torch.arange(3, 3 + batch)
        lens = torch.tensor(own, dtype=torch.int32) + prefix
        o = decoding_attn_paged_shared_prefix_fwd(q.to(DEV), pk.to(DEV), pv.to(DEV), ids, prefix, table.to(DEV), lens.to(DEV), prefix + 2, d, False)
    else:
        o = decoding_attn_shared_prefix_fwd(q.to(DEV), kp.to(DEV), vp.to(DEV), k.to(DEV), v.to(DEV), cu.to(torch.int32).to(DEV), 2, d, False)
    assert torch.isfinite(o).all() and (o != 0).any(-1).all()
    check(o[rows], reference(q[rows], kp, vp, ks, vs, False))


@pytest.mark.parametrize("alibi", [False, True])
def test_a_prefix_past_32_bit_offsets(alibi):
    """More than 2^32 bytes of packed K: the values are zero but in a few tokens near the ends, whose weights a score of 20
    raises far above the others' sum."""
    hk, d, prefix = 32, 128, (1 << 32) // (32 * 128 * 2) + 1000
    g = torch.Generator().manual_seed(40)
    q = torch.zeros(3, hk, d)
    q[:, :, 0] = 1.0
    q = q.half()
    kp = torch.zeros(prefix, hk, d, dtype=torch.float16, device=DEV)
    vp = torch.zeros_like(kp)
    hot = [5, prefix // 2, prefix - 900, prefix - 1]
    top = torch.randn(len(hot), hk, generator=g) + 24.0 * d ** 0.5
    kp[hot, :, 0] = top.half().to(DEV)
    vals = torch.randn(len(hot), hk, d, generator=g).half()
    vp[hot] = vals.to(DEV)
    slopes = torch.full((hk,), 1e-6, device=DEV) if alibi else None
    empty = kp[:0]
    o = decoding_attn_shared_prefix_fwd(q.to(DEV), kp, vp, empty, empty, torch.zeros(4, dtype=torch.int32, device=DEV), 0, d, alibi,
                                        alibi_slopes=slopes)
    x = top.half().double() / d ** 0.5
    if alibi:
        x = x + 1e-6 * (torch.tensor(hot).double() - (prefix - 1))[:, None]
    rest = torch.full((1, hk), math.log(prefix), dtype=torch.float64)  # all other tokens: score 0, value 0
    w = torch.softmax(torch.cat([x, rest]), dim=0)[:-1]
    want = (w[:, :, None] * vals.double()).sum(0)
    # u = 2^-11: u w |v| for the probabilities, as much for the denominator that sums them, u |o| for the result.  The others are
    # e^13.2 against e^23.7 and more, a share below 2^-15, which half precision's probabilities may lose whole
    tol = 2.0 ** -10 * w[:, :, None].mul(vals.double().abs()).sum(0) + (2.0 ** -11 + 2.0 ** -15) * want.abs()
    assert ((o.cpu().double() - want[None]).abs() <= tol[None]).all()


@pytest.mark.parametrize("hq,hk", [(16, 4), (6, 2)])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_weights_rounding_is_in_the_denominator_too(dtype, d, hq, hk):
    """Nearly all the weight on one own token, whose unnormalised probability, some 2^7 of the running maximum's, is rounded
    where a step is largest (1.0 to 1.1 times a power of two): rounded in the sum over V alone it would scale the row by up to half a
    step, beside the result's own, and the values are such that this is a whole one.  (The token lies in the last tile of 129 tokens, so
    that it follows the first tile's maximum in the same wave, also where four waves take tiles in turn, and the batch is large enough
    for sequences that are not split.)"""
    batch, rows = 300, list(range(0, 300, 9))
    g = torch.Generator().manual_seed(d + hq)
    low = -20.0 * d ** 0.5
    q = torch.zeros(batch, hq, d)
    q[:, :, 0] = 1.0
    k = torch.zeros(batch, 129, hk, d)
    k[:, :, :, 0] = low
    k[:, 0, :, 0] = 0.0
    k[:, 128, :, 0] = (7.0 + 0.13 * torch.rand(batch, hk, generator=g)) * math.log(2.0) * d ** 0.5
    v = 1.0 + 0.1 * torch.rand(batch, 129, hk, d, generator=g)
    kp, vp = torch.zeros(1, hk, d), torch.ones(1, hk, d)
    kp[:, :, 0] = low
    q, k, v, kp, vp = (t.to(dtype) for t in (q, k, v, kp, vp))
    ks, vs = list(k), list(v)
    kk, vv, cu, most = packed(ks, vs, hk, d, dtype)
    o = decoding_attn_shared_prefix_fwd(q.to(DEV), kp.to(DEV), vp.to(DEV), kk, vv, cu, most, d, False)
    check(o[rows], some(q, kp, vp, ks, vs, False, rows))
