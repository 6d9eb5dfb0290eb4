"""kv_cache_append and kv_cache_read at the sizes where a work-group takes several turns over its tokens, and whole stores
compared: every byte that is not the call's, the gaps between pages among them, has to stay as it was.

A work-group of 256 threads holds 4 chunks of eight elements a thread (append, quantised: 2 of sixteen) and takes
1024 / (heads * dim / 8) tokens, twice as many from 1024 (append) or 8192 (read) work-groups of K and V together, fewer in small
calls, and at least one, which takes several turns if it is wider.  The definition runs in 64 bits on the GPU here, on all tokens at
once; results are compared for equality, for the reasons given with the small tests.
"""
import pytest
import torch

import kv_cache_oracle as ora
from decoding_attention_amd import kv_cache_append, kv_cache_read

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def bits(t):
    return t.contiguous().view(torch.uint8)


class Store:
    """One plane's pool inside a larger store, random bytes everywhere, with a gap behind each page, and the rows of a call."""

    def __init__(self, g, fmt, dtype, heads, dim, page, pages, tokens, fused):
        self.fmt, self.dtype, self.heads, self.dim, self.page = fmt, dtype, heads, dim, page
        pd = ora.pool_dtype(fmt, dtype)
        self.row = heads * ora.pool_width(fmt, dim) * pd.itemsize  # bytes
        gap = 64 * pd.itemsize
        self.store = torch.randint(0, 256, (pages, page * self.row + gap), generator=g, device=DEV, dtype=torch.uint8)
        if fmt == "fp8":  # (no NaN among what is read back unwritten)
            self.store &= 0x77
        self.before = self.store.clone()
        self.pool = self.rows_of(self.store).unflatten(2, (heads, -1)).view(pd)
        self.scale = None
        if "_" in fmt:
            self.scale = torch.rand(ora.pair_shape(fmt, pages, page, heads, dim), generator=g, device=DEV)
        elif fmt != "16":
            at = {"fp8": 448.0, "int8": 127.0, "int4": 7.0}[fmt]
            self.scale = 4.0 / at * torch.exp(0.5 * torch.randn(heads, generator=g, device=DEV))
        self.scale_before = None if self.scale is None else self.scale.clone()
        x = torch.randn(tokens, heads * (3 if fused else 1), dim, generator=g, device=DEV)
        # a third of the tokens hold few distinct values, whose quotients are often exact half steps
        t = torch.arange(tokens, device=DEV)
        x = torch.where((t % 3 == 0)[:, None, None], torch.round(x * 20) * 0.25, x).to(dtype)
        if fused:
            x = x[:, heads:2 * heads]
        for at, value in ((7, float("nan")), (50, float("inf")), (61, -float("inf"))):  # in some rows of some heads
            x[at::97, heads // 2, (at * 5) % dim] = value
        x[29::101, heads - 1] = 3.0
        self.x = x

    def rows_of(self, store):
        return store[:, :self.page * self.row].unflatten(1, (self.page, self.row))

    def expected(self, pages, rows):
        """What the store and the pairs hold after the call."""
        want, pairs = self.before.clone(), None if self.scale is None else self.scale_before.clone()
        if ora.kind_of(self.fmt) == "16":
            new = bits(self.x).flatten(1)
            pair = None
        else:
            n, pair = ora.quantise(self.x, self.fmt, self.scale_before)
            kind = ora.kind_of(self.fmt)
            if kind == "int4":
                i = n.to(torch.int16) & 15
                new = (i[..., 0::2] | (i[..., 1::2] << 4)).to(torch.uint8).flatten(1)
            else:
                new = bits(n.float().to(torch.float8_e4m3fn) if kind == "fp8" else n.to(torch.int8)).flatten(1)
        self.rows_of(want)[pages, rows] = new
        if pair is not None:
            pairs[pages, rows] = pair
        return want, pairs

    def check(self, pages, rows):
        want, pairs = self.expected(pages, rows)
        got = self.store
        if self.fmt == "fp8":  # (a zero may carry either sign, a NaN as well)
            plain = lambda t: torch.where((t & 0x7F == 0) | (t & 0x7F == 0x7F), t & 0x7F, t)  # noqa: E731
            got, want = plain(got), plain(want)
        assert torch.equal(got, want), f"{int((got != want).sum())} of {got.numel()} bytes differ"
        if pairs is not None:
            same = (self.scale == pairs) | (torch.isnan(self.scale) & torch.isnan(pairs))
            assert same.all(), f"{int((~same).sum())} factors differ"
        elif self.scale is not None:
            assert torch.equal(self.scale, self.scale_before)

    def check_read(self, got, pages, rows):
        held = self.pool.view(torch.uint8)[pages, rows].view(self.pool.dtype)
        n = ora.stored_values(held, self.fmt)
        pair = self.scale[pages, rows] if "_" in self.fmt else None
        want = ora.read_values(n, self.fmt, self.scale, pair, self.dtype)
        plain = lambda t: torch.where(torch.isnan(t), torch.full_like(t, 9.0), t + 0.0)  # noqa: E731  (NaN, -0)
        assert got.shape == want.shape
        assert torch.equal(plain(got), plain(want)), f"{int((plain(got) != plain(want)).sum())} values differ"


def run(fmt, heads, dim, tokens, *, dim_v=None, latent=False, page=16, batch=7, dtype=torch.bfloat16, fused=False, seed=0):
    """Appends `tokens` rows of `batch` ragged sequences, compares the stores, reads the rows back and compares them."""
    g = torch.Generator(DEV).manual_seed(seed)
    gc = torch.Generator().manual_seed(seed)
    cut = torch.sort(torch.randint(0, tokens + 1, (batch - 1,), generator=gc)).values
    cu = torch.cat([torch.zeros(1, dtype=torch.int64), cut, torch.tensor([tokens])])
    new = cu[1:] - cu[:-1]
    lens = new + torch.randint(0, 40, (batch,), generator=gc)
    blocks = (lens + page - 1) // page
    pages = int(blocks.sum()) + 2
    order = torch.randperm(pages, generator=gc)
    table = torch.full((batch, int(blocks.max())), -1, dtype=torch.int64)
    for b, at in enumerate((blocks.cumsum(0) - blocks).tolist()):
        table[b, :blocks[b]] = order[at:at + int(blocks[b])]
    t = torch.arange(tokens)
    b = torch.searchsorted(cu, t, right=True) - 1
    pos = lens[b] - (cu[b + 1] - t)
    in_page, in_row = table[b, pos // page].to(DEV), (pos % page).to(DEV)

    stores = [Store(g, fmt, dtype, heads, dim, page, pages, tokens, fused)]
    if not latent:
        stores.append(Store(g, fmt, dtype, heads, dim_v or dim, page, pages, tokens, fused))
    k, v = stores[0], stores[1] if len(stores) > 1 else None
    args = (k.pool, v.pool if v else None, table.to(torch.int32).to(DEV), lens.to(torch.int32).to(DEV), cu.to(torch.int32).to(DEV))
    scales = dict(k_scale=k.scale, v_scale=v.scale if v else None)
    kv_cache_append(k.x, v.x if v else None, *args, **scales)
    torch.cuda.synchronize()
    for s in stores:
        s.check(in_page, in_row)
        s.before, s.scale_before = s.store.clone(), None if s.scale is None else s.scale.clone()
    got = kv_cache_read(*args, tokens, dtype=dtype, **scales)
    torch.cuda.synchronize()
    for s, o in zip(stores, got):
        s.check_read(o, in_page, in_row)
        assert torch.equal(s.store, s.before)


SOME = ["16", "fp8", "int8", "int4_tok", "int8_g64"]


@pytest.mark.parametrize("tokens", [500, 4088, 4093, 32773])
@pytest.mark.parametrize("fmt", ora.FORMATS)
def test_several_turns_of_a_work_group(fmt, tokens):
    """32 heads d 64, four tokens a work-group, eight from 4089 tokens (append) or 32761 (read); the last one is cut short."""
    run(fmt, 32, 64, tokens, seed=tokens, dtype=torch.float16 if tokens == 4093 else torch.bfloat16)


@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("fmt", SOME)
def test_two_turns_with_odd_heads(fmt, fused):
    """5 heads d 128: chunks that are no power of two, 12 tokens a work-group and 24 in this call."""
    run(fmt, 5, 128, 12297, fused=fused, page=64, batch=300, seed=3)


@pytest.mark.parametrize("fmt", SOME)
def test_a_hundred_and_twenty_eight_tokens_a_work_group(fmt):
    """2 heads d 64, 64 tokens a work-group and 128, the most there are, in this call."""
    run(fmt, 2, 64, 65536 + 11, page=1, batch=3, seed=4)


@pytest.mark.parametrize("fmt", ora.FORMATS)
@pytest.mark.parametrize("heads,dim", [(64, 256), (33, 256), (130, 128), (257, 64)])
def test_a_token_wider_than_a_turn(heads, dim, fmt):
    """One token a work-group, several turns of it."""
    run(fmt, heads, dim, 70, page=8, batch=4, seed=heads)


@pytest.mark.parametrize("fmt", ["16", "fp8", "int8", "int4"])
def test_rows_of_96(fmt):
    run(fmt, 4, 96, 21600, page=32, seed=5)


@pytest.mark.parametrize("tokens", [1, 90, 28700])
@pytest.mark.parametrize("fmt", ["16", "fp8", "int8", "int4"])
def test_latent_rows_alone_and_with_values_of_their_own(fmt, tokens):
    """(576, 512): V inside K, and in a pool of its own, whose rows are narrower than K's."""
    run(fmt, 1, 576, tokens, latent=True, page=64, batch=3, seed=tokens)
    for heads in (1, 3):
        run(fmt, heads, 576, min(tokens, 15000), dim_v=512, page=64, batch=3, seed=tokens + heads)


@pytest.mark.parametrize("page", [1, 2, 16, 256])
@pytest.mark.parametrize("fmt", ora.FORMATS)
def test_gaps_between_pages_stay_as_they_were(fmt, page):
    run(fmt, 3, 128, 333, page=page, batch=5, seed=page)


@pytest.mark.parametrize("fmt", ["16", "int8_tok"])
@pytest.mark.parametrize("batch", [513, 5000, 70001])
def test_thousands_of_sequences(fmt, batch):
    """More sequences than marks, most of them without a row in the call: the second search is many steps long."""
    run(fmt, 2, 64, 3001, batch=batch, seed=batch)
