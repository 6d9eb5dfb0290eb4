"""K/V rows written into a paged cache and read back (kv_cache_append, kv_cache_read) against the definition in 64 bits.

What an append stores is a whole number of the format, a float32 pair, or a copy: it is compared for equality.  So is what a
read returns: both sides round once per float32 operation and once to 16 bits.
"""
import pytest
import torch

import kv_cache_oracle as ora
from decoding_attention_amd import decoding_attn_fwd, decoding_attn_paged_fwd, kv_cache_append, kv_cache_read
from decoding_attention_amd import workloads as wl

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


class Cache:
    """A cache with its block table, every unused byte marked, and the call's rows, on the CPU and on the GPU."""

    def __init__(self, fmt, dtype, heads, dim, page, lens, new, *, latent=False, seed=0, stride_pages=False, scales=True,
                 table_cols=0):
        g = torch.Generator().manual_seed(seed)
        self.fmt, self.dtype, self.heads, self.page, self.lens = fmt, dtype, heads, page, list(lens)
        blocks = [(n + page - 1) // page for n in lens]
        self.pages = sum(blocks) + 2
        order = torch.randperm(self.pages, generator=g).tolist()
        self.table = torch.full((len(lens), max(1, max(blocks), table_cols)), -1, dtype=torch.int32)
        for b, n in enumerate(blocks):
            for i in range(n):
                self.table[b, i] = order.pop()
        self.cu = None if new is None else torch.tensor([0] + list(torch.tensor(new).cumsum(0)), dtype=torch.int32)
        self.tokens = len(lens) if new is None else int(self.cu[-1])
        self.names = ["k"] if latent else ["k", "v"]
        self.dims = {"k": dim, "v": dim}
        self.pool, self.dpool, self.scale, self.dscale, self.x = {}, {}, {"k": None, "v": None}, {"k": None, "v": None}, {}
        for nm in self.names:
            d = self.dims[nm]
            width = ora.pool_width(fmt, d)
            wide = (2 if stride_pages else 1) * page * heads * width
            store = torch.randint(0, 120, (self.pages, wide), generator=g, dtype=torch.int16)
            pd = ora.pool_dtype(fmt, dtype)
            store = store.to(torch.uint8).view(pd) if pd.itemsize == 1 else store.to(pd)
            cut = lambda t: t[:, :page * heads * width].unflatten(1, (page, heads, width))  # noqa: E731
            self.pool[nm], self.dpool[nm] = cut(store), cut(store.to(DEV))
            self.whole = store
            if fmt == "16":
                pass
            elif "_" in fmt:
                s = torch.rand(ora.pair_shape(fmt, self.pages, page, heads, d), generator=g)
                self.scale[nm], self.dscale[nm] = s, s.to(DEV)
            elif scales:
                at = {"fp8": 448.0, "int8": 127.0, "int4": 7.0}[fmt]
                s = 4.0 / at * torch.exp(0.5 * torch.randn(heads, generator=g))
                self.scale[nm], self.dscale[nm] = s, s.to(DEV)
            self.x[nm] = torch.randn(self.tokens, heads, d, generator=g).to(dtype)
        self.at = ora.places(self.table, self.lens, None if self.cu is None else self.cu.tolist(), self.tokens, page,
                             self.pages)

    def gpu_args(self):
        return (self.dpool["k"], self.dpool.get("v"), self.table.to(DEV), torch.tensor(self.lens, dtype=torch.int32, device=DEV),
                None if self.cu is None else self.cu.to(DEV))

    def append(self, dx=None):
        dx = dx or {n: x.to(DEV) for n, x in self.x.items()}
        pk, pv, t, ln, cu = self.gpu_args()
        kv_cache_append(dx["k"], dx.get("v"), pk, pv, t, ln, cu, k_scale=self.dscale["k"], v_scale=self.dscale["v"])
        torch.cuda.synchronize()

    def read(self, **kw):
        pk, pv, t, ln, cu = self.gpu_args()
        out = kv_cache_read(pk, pv, t, ln, cu, self.tokens, dtype=self.dtype, k_scale=self.dscale["k"],
                            v_scale=self.dscale["v"], **kw)
        torch.cuda.synchronize()
        return out

    def expected(self):
        """Applies the append to the CPU's copy of the pools and pairs."""
        for nm in self.names:
            n, pair = ora.quantise(self.x[nm], self.fmt, self.scale[nm])
            kind = ora.kind_of(self.fmt)
            if kind == "int4":
                i = n.to(torch.int16) & 15
                rows = (i[..., 0::2] | (i[..., 1::2] << 4)).to(torch.uint8)
            elif kind == "fp8":
                rows = n.float().to(torch.float8_e4m3fn)
            else:  # (a 16-bit row is a copy, bit for bit: a NaN keeps its payload)
                rows = self.x[nm] if kind == "16" else n.to(self.pool[nm].dtype)
            for t, at in enumerate(self.at):
                if isinstance(at, tuple):
                    bits = ora.INT_OF.get(rows.dtype, rows.dtype)
                    self.pool[nm].view(bits)[at[0], at[1]] = rows.view(bits)[t]
                    if pair is not None:
                        self.scale[nm][at[0], at[1]] = pair[t]

    def check_pools(self):
        for nm in self.names:
            got, want = self.dpool[nm].cpu(), self.pool[nm]
            if got.dtype == torch.float8_e4m3fn:  # (a zero may carry either sign)
                got, want = got.float(), want.float()
                assert torch.equal(torch.isnan(got), torch.isnan(want))
                got, want = got.nan_to_num(7.0), want.nan_to_num(7.0)
            elif got.dtype in ora.INT_OF:
                got, want = got.view(torch.int16), want.view(torch.int16)
            assert torch.equal(got, want), f"{nm}: {(got != want).sum()} of {got.numel()} stored values differ"
            if self.scale[nm] is not None:
                a, b = self.dscale[nm].cpu(), self.scale[nm]
                assert torch.equal(a.view(torch.int32), b.view(torch.int32)) or (
                    torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a.nan_to_num(1.0), b.nan_to_num(1.0)))

    def check_read(self, got, before=None):
        for nm, o in zip(self.names, got):
            o = o.cpu()
            rows, pairs = [], []
            for at in self.at:
                rows.append(self.pool[nm][at] if isinstance(at, tuple) else torch.zeros_like(self.pool[nm][0, 0]))
                if "_" in self.fmt:
                    pairs.append(self.scale[nm][at] if isinstance(at, tuple) else torch.zeros_like(self.scale[nm][0, 0]))
            n = ora.stored_values(torch.stack(rows), self.fmt)
            want = ora.read_values(n, self.fmt, self.scale[nm], torch.stack(pairs) if pairs else None, self.dtype)
            for t, at in enumerate(self.at):
                if at is None:
                    want[t] = 0
                elif at == "behind":
                    want[t] = before[t] if before is not None else o[t]
            bits = (lambda t: torch.where(torch.isnan(t), torch.full_like(t, 9.0), t + 0.0))  # (NaN, -0)
            assert torch.equal(bits(o), bits(want)), f"{nm}: {(bits(o) != bits(want)).sum()} values differ"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("fmt", ora.FORMATS)
def test_append_and_read(fmt, dim, dtype):
    if "_" in fmt and dim == 96:
        pytest.skip("pairs: 64, 128, 256")
    c = Cache(fmt, dtype, 3, dim, 16, [1, 40, 16, 0, 33, 17], [1, 7, 16, 0, 33, 2], seed=dim)
    c.append()
    c.expected()
    c.check_pools()
    c.check_read(c.read())


@pytest.mark.parametrize("page", [1, 2, 64, 1024])
@pytest.mark.parametrize("fmt", ["16", "int4_tok", "fp8"])
def test_page_sizes_heads_and_strides_between_pages(fmt, page):
    for heads in (1, 5, 32):
        c = Cache(fmt, torch.bfloat16, heads, 128, page, [70, 3, 129], [5, 3, 129], seed=page + heads, stride_pages=True)
        c.append()
        c.expected()
        c.check_pools()
        c.check_read(c.read())


@pytest.mark.parametrize("fmt", ["16", "int8", "int8_g64"])
def test_one_token_per_sequence_and_padded_rows(fmt):
    """A decode step: no cu_seq; sequences of length 0 are rows of the batch without a sequence."""
    c = Cache(fmt, torch.float16, 8, 128, 16, [5, 0, 16, 17, 1, 0, 300], None, seed=3)
    c.append()
    c.expected()
    c.check_pools()
    c.check_read(c.read())


@pytest.mark.parametrize("batch", [1, 2, 63, 64, 65, 255, 256, 257, 300])
def test_many_sequences_with_empty_ones_between(batch):
    g = torch.Generator().manual_seed(batch)
    new = torch.randint(0, 4, (batch,), generator=g)
    new[0] = 2
    lens = new + torch.randint(0, 40, (batch,), generator=g)
    c = Cache("int4_tok", torch.bfloat16, 2, 64, 16, lens.tolist(), new.tolist(), seed=batch)
    c.append()
    c.expected()
    c.check_pools()
    c.check_read(c.read())


@pytest.mark.parametrize("fmt", ["16", "fp8", "int8", "int4"])
def test_latent_rows(fmt):
    """(576, 512): one row holds K and V."""
    c = Cache(fmt, torch.bfloat16, 1, 576, 64, [100, 64, 1], [40, 64, 1], latent=True, seed=5)
    c.append()
    c.expected()
    c.check_pools()
    k, v = c.read()
    assert v is None
    c.check_read([k])


@pytest.mark.parametrize("fmt", ["fp8", "int8", "int4"])
def test_factors_default_to_one(fmt):
    c = Cache(fmt, torch.float16, 2, 64, 16, [20], [20], scales=False, seed=6)
    for nm in c.names:
        c.x[nm] = (c.x[nm].float() * 40).to(torch.float16)  # (beyond int4's range: clamped)
    c.append()
    c.expected()
    c.check_pools()
    c.check_read(c.read())


@pytest.mark.parametrize("fmt", ["fp8", "int8", "int8_g64", "int4_tok", "16"])
@pytest.mark.parametrize("cut", ["fused", "odd", "expanded"])
def test_strided_rows(fmt, cut):
    """k and v as columns of a fused projection's output, at addresses that are no multiple of 16 bytes, and one row for
    every head."""
    c = Cache(fmt, torch.bfloat16, 4, 64, 16, [50, 9], [31, 9], seed=8)
    g = torch.Generator().manual_seed(9)
    dx = {}
    for nm in c.names:
        if cut == "fused":
            x = torch.randn(c.tokens, 12, 64, generator=g).to(torch.bfloat16).to(DEV)[:, 4:8]
        elif cut == "odd":
            x = torch.randn(c.tokens, 4 * 64 + 3, generator=g).to(torch.bfloat16).to(DEV)[:, 1:257].unflatten(1, (4, 64))
        else:
            x = torch.randn(c.tokens, 1, 64, generator=g).to(torch.bfloat16).to(DEV).expand(-1, 4, -1)
        dx[nm], c.x[nm] = x, x.cpu().contiguous()
    c.append(dx)
    c.expected()
    c.check_pools()


def test_ties_go_to_even_and_saturate():
    """Values that lie exactly half-way between two steps, the largest and the infinite ones."""
    vals = [0.5, 1.5, 2.5, -0.5, -1.5, 3.5, 6.5, 7.5, -7.5, -8.5, 126.5, 127.5, -127.5, -128.5, 300.0, -300.0, 448.0, 464.0,
            480.0, 1000.0, float("inf"), -float("inf"), 17.0, 19.0, 2.0 ** -10, 3 * 2.0 ** -10, 2.0 ** -11, 0.0, 5 * 2.0 ** -10, 9.0,
            2.0 ** -7 + 2.0 ** -10, 1.0625]
    for fmt in ("fp8", "int8", "int4"):
        c = Cache(fmt, torch.float16, 1, 64, 16, [1], [1], scales=False)
        for nm in c.names:
            c.x[nm] = torch.tensor(vals + [-v for v in vals]).view(1, 1, 64).half()
        c.append()
        c.expected()
        c.check_pools()


@pytest.mark.parametrize("fmt", ora.FORMATS[1:])
def test_small_whole_numbers_and_constant_rows(fmt):
    """Rows of few distinct values: their quotients are often exact half steps.  A constant row has the least scale."""
    c = Cache(fmt, torch.bfloat16, 2, 128, 16, [64], [64], seed=11)
    g = torch.Generator().manual_seed(12)
    for nm in c.names:
        x = torch.randint(-60, 60, (64, 2, 128), generator=g).float() * 0.25
        x[0], x[1], x[2, :, :64], x[3] = 0.0, 3.0, -7.0, 1e-30
        c.x[nm] = x.to(torch.bfloat16)
    c.append()
    c.expected()
    c.check_pools()
    c.check_read(c.read())


@pytest.mark.parametrize("fmt", ora.FORMATS)
def test_nan_and_infinite_values(fmt):
    c = Cache(fmt, torch.bfloat16, 2, 128, 16, [8], [8], seed=13)
    for nm in c.names:
        c.x[nm][1, 0, 5] = float("nan")
        c.x[nm][2, 1, 127] = float("inf")
        c.x[nm][3, 0, 64] = -float("inf")
        c.x[nm][4, 1] = float("nan")
        if fmt != "16":
            c.x[nm][0, 1, 3] = 3e38
    c.append()
    c.expected()
    c.check_pools()
    if "_" not in fmt:
        c.check_read(c.read())
    else:
        got = c.read()[0].cpu()
        run = slice(0, 64) if fmt.endswith("g64") else slice(0, 128)
        assert torch.isnan(got[1, 0, run]).all() and torch.isnan(got[4, 1]).all()
        assert torch.isfinite(got[5:]).all() and torch.isfinite(got[0, 0]).all()


def test_tokens_without_a_place_are_skipped():
    """Page ids outside the pools, positions behind the block table, lengths below the number of new tokens, rows behind the
    last sequence: nothing is written for them, and they read as zeros (the last: left as they were)."""
    c = Cache("int8_tok", torch.float16, 2, 64, 16, [40, 20, 3, 33], [40, 20, 3, 33], seed=14)
    c.table[0, 1] = -1
    c.table[1, 0] = c.pages
    c.lens[2] = 1          # its first two tokens would lie before the sequence
    c.lens[3] = 33 + 48    # three tables' worth of pages: the row of the table ends before them
    extra = 5              # rows behind cu_seq[batch]
    c.tokens += extra
    g = torch.Generator().manual_seed(15)
    for nm in c.names:
        c.x[nm] = torch.randn(c.tokens, 2, 64, generator=g).half()
    c.at = ora.places(c.table, c.lens, c.cu.tolist(), c.tokens, c.page, c.pages)
    assert c.at.count(None) > 30 and c.at.count("behind") == extra
    c.append()
    c.expected()
    c.check_pools()
    mark = {nm: torch.full((c.tokens, 2, 64), 5.5, dtype=torch.float16, device=DEV) for nm in c.names}
    got = c.read(k_out=mark["k"], v_out=mark["v"])
    assert got[0].data_ptr() == mark["k"].data_ptr()
    c.check_read(got, before=torch.full((c.tokens, 2, 64), 5.5, dtype=torch.float16))


def test_no_tokens():
    c = Cache("int8", torch.float16, 2, 64, 16, [40, 20], [0, 0], seed=16)
    c.append()
    c.check_pools()
    k, v = c.read()
    assert tuple(k.shape) == (0, 2, 64) and tuple(v.shape) == (0, 2, 64)


def test_offsets_past_32_bits():
    """A pool of more than 4 GiB and more than 2^31 elements: the last pages are the right ones."""
    heads, dim, page = 8, 128, 256
    pages = (1 << 32) // (page * heads * dim * 2) + 8
    pool = torch.zeros((pages, page, heads, dim), dtype=torch.float16, device=DEV)
    table = torch.tensor([[pages - 1, 3], [pages - 2, pages - 3]], dtype=torch.int32, device=DEV)
    lens = torch.tensor([300, 512], dtype=torch.int32, device=DEV)
    cu = torch.tensor([0, 100, 612], dtype=torch.int32, device=DEV)
    x = torch.randn(612, heads, dim, device=DEV).half()
    kv_cache_append(x, x, pool, pool.clone(), table, lens, cu)
    assert torch.equal(pool[pages - 1, 200:], x[:56]) and torch.equal(pool[3, :44], x[56:100])
    assert torch.equal(pool[pages - 2], x[100:356]) and torch.equal(pool[pages - 3], x[356:])
    assert int((pool != 0).any(-1).any(-1).sum()) == 612
    k, _ = kv_cache_read(pool, pool, table, lens, cu, 612, dtype=torch.float16)
    assert torch.equal(k, x)


def test_other_streams_and_replays():
    """Append and read on a stream of their own, then captured and replayed on changed rows and lengths."""
    c = Cache("int4_g64", torch.bfloat16, 4, 128, 16, [64, 64, 64], None, seed=17, table_cols=4)
    pk, pv, table, lens, _ = c.gpu_args()
    k = torch.empty(3, 4, 128, dtype=torch.bfloat16, device=DEV)
    v = torch.empty_like(k)

    def step():
        kv_cache_append(k, v, pk, pv, table, lens, k_scale=c.dscale["k"], v_scale=c.dscale["v"])
        return kv_cache_read(pk, pv, table, lens, None, 3, dtype=torch.bfloat16, k_scale=c.dscale["k"], v_scale=c.dscale["v"])

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        k.copy_(c.x["k"])
        v.copy_(c.x["v"])
        step()
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    g = torch.Generator().manual_seed(18)
    for length in (64, 1, 17, 33):
        c.lens = [length, 64 - length, length]
        lens.copy_(torch.tensor(c.lens, dtype=torch.int32))
        for nm, t in (("k", k), ("v", v)):
            c.x[nm] = torch.randn(3, 4, 128, generator=g).to(torch.bfloat16)
            t.copy_(c.x[nm])
        graph.replay()
        torch.cuda.synchronize()
        c.at = ora.places(c.table, c.lens, None, 3, c.page, c.pages)
        for nm in c.names:
            c.pool[nm].copy_(c.dpool[nm].cpu()), c.scale[nm].copy_(c.dscale[nm].cpu())
        c.expected()
        c.check_pools()
        c.check_read([t.clone() for t in out])


@pytest.mark.parametrize("fmt,dtype", [("16", torch.float16), ("fp8", torch.bfloat16), ("int8", torch.bfloat16),
                                       ("int4", torch.float16), ("int4_tok", torch.bfloat16), ("int8_g64", torch.float16)])
def test_attention_over_an_appended_cache(fmt, dtype):
    """Prompt and decode steps appended, the attention over the pages, and the same attention over what a read returns: both
    see the same cache, so they differ by the roundings of the read rows to 16 bits and the two products' probabilities."""
    w = wl.make_workload(5, 8, 4, 128, 128, 300, dtype, seed=20, varlen=True, min_len=4)
    lens = torch.tensor(w.lengths, dtype=torch.int32)
    c = Cache(fmt, dtype, 4, 128, 16, w.lengths, (lens - 3).tolist(), seed=21)
    cu_all = w.cu_seq_k.tolist()
    # the prompts first (all but three tokens of each sequence), then three steps of one token
    for nm, src in (("k", w.k), ("v", w.v)):
        c.x[nm] = torch.cat([src[cu_all[b]:cu_all[b + 1] - 3] for b in range(5)])
    c.lens = (lens - 3).tolist()
    c.append()
    c.cu, c.tokens = None, 5
    for step in range(3):
        for nm, src in (("k", w.k), ("v", w.v)):
            c.x[nm] = torch.stack([src[cu_all[b + 1] - 3 + step] for b in range(5)])
        c.lens = (lens - 2 + step).tolist()
        c.append()
    q, ln = w.q.to(DEV), lens.to(DEV)
    paged = decoding_attn_paged_fwd(q, c.dpool["k"], c.dpool["v"], c.table.to(DEV), ln, w.max_seq_k, 128, False,
                                    k_scale=c.dscale["k"], v_scale=c.dscale["v"])
    k, v = kv_cache_read(c.dpool["k"], c.dpool["v"], c.table.to(DEV), ln, w.cu_seq_k.to(DEV), int(cu_all[-1]), dtype=dtype,
                         k_scale=c.dscale["k"], v_scale=c.dscale["v"])
    packed = decoding_attn_fwd(q, k, v, w.cu_seq_k.to(DEV), w.max_seq_k, 128, False)
    # a score changes by at most u |q|.|k| scale (u half a step), its weight by that much relative; V and the two results by
    # u each; the probabilities of either product by u
    u = torch.finfo(dtype).eps / 2
    big = float(v.float().abs().max())
    move = u * float((w.q.float().abs().amax(dim=(1, 2)).max() * k.float().abs().sum(-1).max())) / 128 ** 0.5
    assert (paged.float() - packed.float()).abs().max().item() <= (2 * move + 5 * u) * big
    if fmt == "16":
        assert torch.equal(k.cpu().view(torch.int16), w.k.view(torch.int16))


@pytest.mark.parametrize("fmt", ["16", "fp8", "int8_g64", "int4_tok"])
@pytest.mark.parametrize("extra", [1, 70, 1 << 22])
def test_rows_behind_the_last_sequence_need_not_be_there(fmt, extra):
    """The C call with a count beyond cu_seq[batch] (a captured graph's largest step): k and v hold the sequences' rows alone."""
    from decoding_attention_amd import _lib
    lib = _lib.load()
    c = Cache(fmt, torch.bfloat16, 4, 128, 16, [50, 0, 9], [31, 0, 9], seed=30)
    dx = {n: x.to(DEV) for n, x in c.x.items()}
    pk, pv, table, lens, cu = c.gpu_args()
    pack = 2 if fmt.startswith("int4") else 1
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    forms = {"16": (0, 0), "fp8": (1, 0), "int8_g64": (2, 2), "int4_tok": (3, 1)}[fmt]
    rc = lib.da_kv_cache_append(dx["k"].data_ptr(), dx["v"].data_ptr(), 512, 128, 512, 128, pk.data_ptr(), pv.data_ptr(),
                                table.data_ptr(), lens.data_ptr(), cu.data_ptr(), c.tokens + extra, 3, 4, 128, 128, 16,
                                table.shape[1], c.pages, pk.stride(0) * pack, pv.stride(0) * pack, 1, *forms, ptr(c.dscale["k"]),
                                ptr(c.dscale["v"]), torch.cuda.current_stream().cuda_stream)
    assert rc == 0, _lib.last_error()
    torch.cuda.synchronize()
    c.expected()
    c.check_pools()


def test_replays_of_a_padded_append():
    """One captured call for steps of up to 96 rows: cu_seq on the device says how many there are, the rows behind hold NaN."""
    c = Cache("int8_tok", torch.bfloat16, 2, 64, 16, [96, 96], [48, 48], seed=31)
    pk, pv, table, lens, cu = c.gpu_args()
    k = torch.full((96, 2, 64), float("nan"), dtype=torch.bfloat16, device=DEV)
    v = k.clone()

    def step():
        kv_cache_append(k, v, pk, pv, table, lens, cu, k_scale=c.dscale["k"], v_scale=c.dscale["v"])

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    g = torch.Generator().manual_seed(32)
    for a, b in ((48, 48), (1, 0), (0, 33), (0, 0), (17, 2)):
        c.cu = torch.tensor([0, a, a + b], dtype=torch.int32)
        c.lens, c.tokens = [96 - a, 40 + b], a + b
        cu.copy_(c.cu), lens.copy_(torch.tensor(c.lens, dtype=torch.int32))
        for nm, t in (("k", k), ("v", v)):
            c.x[nm] = torch.randn(a + b, 2, 64, generator=g).to(torch.bfloat16)
            t.fill_(float("nan"))
            t[:a + b].copy_(c.x[nm])
        for nm in c.names:
            c.pool[nm].copy_(c.dpool[nm].cpu()), c.scale[nm].copy_(c.dscale[nm].cpu())
        graph.replay()
        torch.cuda.synchronize()
        c.at = ora.places(c.table, c.lens, c.cu.tolist(), a + b, c.page, c.pages)
        if a + b:
            c.expected()
        c.check_pools()
