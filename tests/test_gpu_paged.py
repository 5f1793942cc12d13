"""The paged cache on the GPU: attention over it, in rows and in MXFP4, and the appending ops.

Attention is held to the bound that tests/_paged.py derives from the roundings; the 4-bit cache's
codes, scales and values have to be equal to the bit.
"""

import math

import pytest
import torch

from popcorn_amd import _lib, impls
from popcorn_amd.compat import references as R
from tests._paged import HALF_STEP, cache_of, check, exact, mxfp4_of, table_of, values_of

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
INF, NAN = math.inf, math.nan


@pytest.fixture(scope="module", autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")


@pytest.fixture(autouse=True, params=["", "long-table"])
def _long_table(request, monkeypatch):
    """Every packed call also with a table that has room for 2^21 keys, which selects the kernel of many rows where a
    sequence has more than 32 (and lets any call split its keys): the entries behind the test's are outside the pool."""
    if not request.param:
        return

    def longer(op, at):
        def call(*args, **kwargs):
            args = list(args)
            if len(args) > at + 2 and args[at + 2] is not None and args[at].dim() == 2:
                room = (1 << 21) // max(args[1].shape[2], 16) - args[at].shape[1]
                args[at] = torch.nn.functional.pad(args[at], (0, max(room, 0)), value=-1)
            return op(*args, **kwargs)
        return call

    monkeypatch.setattr(impls, "attn_paged", longer(impls.attn_paged, 3))
    monkeypatch.setattr(impls, "attn_paged_mxfp4", longer(impls.attn_paged_mxfp4, 5))


def _run(lens, news, hq, hkv, d, ps, dtype, mxfp4=False, causal=True, scale=None, seed=0, spare=3, width=None, packed=None,
         table=None):
    """One call against float64. news None: one token each, without offsets."""
    need = sum(-(-n // ps) for n in lens) + spare
    cache = cache_of(need, hkv, ps, d, dtype, seed)
    width = max(1, max(-(-n // ps) for n in lens)) if width is None else width
    table = table_of(lens, ps, need, width, seed + 1) if table is None else table
    cu = None
    if news is not None:
        cu = torch.tensor([0, *torch.tensor(news).cumsum(0).tolist()], dtype=torch.int32)
    total = len(lens) if news is None else sum(news)
    q = torch.randn(total, hq, d, generator=torch.Generator().manual_seed(seed + 2)).to(dtype)
    lens_t = torch.tensor(lens, dtype=torch.int32)
    common = (table.to(DEV), lens_t.to(DEV), None if cu is None else cu.to(DEV), causal, scale)
    if mxfp4:
        held = [mxfp4_of(c) for c in cache]
        rows = [values_of(*h) for h in held]
        got = impls.attn_paged_mxfp4(q.to(DEV), *(t.to(DEV) for h in held for t in h), *common)
    else:
        rows = cache
        got = impls.attn_paged(q.to(DEV), *(c.to(DEV) for c in cache), *common)
    torch.cuda.synchronize()
    assert got.shape == q.shape and got.dtype == dtype
    check(got, exact(q, *rows, table, lens, cu, causal, scale), dtype, d, max(lens), mxfp4,
          f"lens {lens} news {news} {hq}/{hkv} x {d} page {ps} {dtype} mxfp4={mxfp4}")
    return got


@pytest.mark.parametrize("dtype", [BF, F16, F32], ids=str)
@pytest.mark.parametrize("mxfp4", [False, True], ids=["rows", "mxfp4"])
def test_one_token_over_lengths(dtype, mxfp4):
    """Every length around a tile, a step, a page and a chunk, none among them."""
    _run([0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 511, 512, 513, 1100], None, 8, 2, 128, 16, dtype, mxfp4)


@pytest.mark.parametrize("d", [8, 16, 40, 64, 72, 80, 96, 128, 136, 192, 200, 256])
@pytest.mark.parametrize("dtype", [BF, F16, F32], ids=str)
def test_head_dims(d, dtype):
    _run([70, 33], None, 4, 2, d, 16, dtype)
    _run([90, 41], [40, 3], 4, 2, d, 32, dtype)


@pytest.mark.parametrize("d", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("dtype", [BF, F16, F32], ids=str)
def test_head_dims_mxfp4(d, dtype):
    _run([70, 133], None, 4, 2, d, 16, dtype, True)
    _run([90, 141], [40, 3], 4, 2, d, 32, dtype, True)


@pytest.mark.parametrize("mxfp4", [False, True], ids=["rows", "mxfp4"])
@pytest.mark.parametrize("heads", [(1, 1), (3, 1), (7, 1), (5, 5), (12, 4), (16, 1), (17, 1), (40, 2), (64, 1)], ids=str)
def test_groups(heads, mxfp4):
    _run([100, 37, 260], None, *heads, 64, 16, BF, mxfp4)
    _run([100, 37, 260], [5, 37, 90], *heads, 64, 16, BF, mxfp4)


@pytest.mark.parametrize("mxfp4", [False, True], ids=["rows", "mxfp4"])
@pytest.mark.parametrize("ps", [16, 48, 80, 128, 256])
def test_page_sizes(ps, mxfp4):
    _run([300, 17, 255, 256], None, 8, 2, 64, ps, BF, mxfp4)
    _run([300, 17, 255, 256], [130, 2, 1, 100], 8, 2, 64, ps, F16, mxfp4)


@pytest.mark.parametrize("mxfp4", [False, True], ids=["rows", "mxfp4"])
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
@pytest.mark.parametrize("dtype", [BF, F32], ids=str)
def test_runs_of_new_tokens(causal, mxfp4, dtype):
    """Sequences without new tokens, whole prompts, chunks, more new tokens than keys (their first see nothing)."""
    _run([50, 64, 200, 9, 333], [0, 64, 70, 12, 1], 4, 2, 64, 16, dtype, mxfp4, causal)
    _run([700], [300], 8, 2, 128, 64, dtype, mxfp4, causal)


@pytest.mark.parametrize("mxfp4", [False, True], ids=["rows", "mxfp4"])
@pytest.mark.parametrize("news", [None, [1, 3], [40, 60]], ids=str)
def test_split_keys(news, mxfp4):
    """Long sequences beside short ones: chunks joined by the second kernel."""
    _run([5000, 90], news, 8, 2, 64, 32, BF, mxfp4)
    _run([3100, 2049], news, 4, 4, 128, 16, F32, mxfp4, scale=0.3)


@pytest.mark.parametrize("mxfp4", [False, True], ids=["rows", "mxfp4"])
@pytest.mark.parametrize("dtype", [BF, F16, F32], ids=str)
def test_many_row_tiles(dtype, mxfp4):
    """512 blocks of 128 rows and more: one round of them, whose keys stay whole."""
    _run([150, 40], [130, 2], 512, 64, 32, 16, dtype, mxfp4)
    _run([70, 33], [35, 33], 1024, 64, 96, 16, dtype, mxfp4)


def test_many_sequences():
    """More than a wave looks at together, lengths of every kind; a scale that is negative."""
    lens = [(37 * i) % 150 for i in range(150)]
    _run(lens, None, 4, 2, 32, 16, BF)
    _run(lens, [min(n, i % 4) for i, n in enumerate(lens)], 4, 2, 32, 16, F16, scale=-0.2)
    _run([3 * n for n in lens], None, 2, 2, 64, 16, BF, True, width=64)


@pytest.mark.parametrize("mxfp4", [False, True], ids=["rows", "mxfp4"])
def test_table_entries_outside_the_pool_are_left_out(mxfp4):
    lens, ps = [200, 40, 33], 16
    table = table_of(lens, ps, 30, 16, 5)
    table[0, 1] = -1
    table[0, 7] = 30
    table[0, 12] = 2 ** 31 - 1
    table[1, :] = -1  # no key at all: zeros
    table[2, 2] = -7  # the page that ends with the newest key
    got = _run(lens, None, 4, 2, 64, ps, BF, mxfp4, table=table, spare=30 - sum(-(-n // ps) for n in lens))
    assert torch.equal(got[1], torch.zeros_like(got[1]))
    _run(lens, [40, 40, 2], 4, 2, 64, ps, F32, mxfp4, table=table, spare=30 - sum(-(-n // ps) for n in lens))


def test_lengths_outside_the_table_are_cut():
    lens = [10_000, -4, 64]
    cache = cache_of(8, 1, 16, 64, BF, 3)
    table = torch.tensor([[0, 1, 2, 3], [1, 2, 3, 4], [4, 5, 6, 7]], dtype=torch.int32)
    q = torch.randn(3, 2, 64).to(BF)
    got = impls.attn_paged(q.to(DEV), *(c.to(DEV) for c in cache), table.to(DEV), torch.tensor(lens, dtype=torch.int32).to(DEV))
    check(got, exact(q, *cache, table, lens, None, True, None), BF, 64, 64)
    assert torch.equal(got[1], torch.zeros_like(got[1]))


def test_tokens_of_no_sequence_are_zeros():
    """A padded batch: offsets that end before the last token, and start behind the first."""
    cache = cache_of(8, 2, 16, 64, BF, 3)
    table = torch.arange(8, dtype=torch.int32).view(2, 4)
    lens = torch.tensor([50, 60], dtype=torch.int32)
    q = torch.randn(70, 4, 64, generator=torch.Generator().manual_seed(1)).to(BF)
    cu = torch.tensor([3, 10, 40], dtype=torch.int32)
    got = impls.attn_paged(q.to(DEV), *(c.to(DEV) for c in cache), table.to(DEV), lens.to(DEV), cu.to(DEV)).cpu()
    alone = impls.attn_paged(q[3:40].to(DEV), *(c.to(DEV) for c in cache), table.to(DEV), lens.to(DEV), (cu - 3).to(DEV)).cpu()
    assert torch.equal(got[3:40], alone)
    assert not got[:3].any() and not got[40:].any()


@pytest.mark.parametrize("dtype", [BF, F16, F32], ids=str)
@pytest.mark.parametrize("news", [None, [1, 1, 1], [20, 30, 9]], ids=str)
def test_what_lies_behind_the_keys_is_not_looked_at(dtype, news):
    """NaN and Inf in every cache row that no sequence has a key in, and in pages no table names."""
    lens, ps, d = [37, 100, 9], 32, 64
    cache = cache_of(12, 2, ps, d, dtype, 9)
    table = table_of(lens, ps, 12, 4, 10)
    mine = torch.zeros(12, ps, dtype=torch.bool)
    for i, n in enumerate(lens):
        for j in range(n):
            mine[table[i, j // ps], j % ps] = True
    total = 3 if news is None else sum(news)
    q = torch.randn(total, 4, d, generator=torch.Generator().manual_seed(2)).to(dtype).to(DEV)
    cu = None if news is None else torch.tensor([0, *torch.tensor(news).cumsum(0).tolist()], dtype=torch.int32).to(DEV)
    rest = (table.to(DEV), torch.tensor(lens, dtype=torch.int32).to(DEV), cu)
    clean = impls.attn_paged(q, *(c.to(DEV) for c in cache), *rest)
    dirty = [c.masked_fill(~mine[:, None, :, None], bad) for c, bad in zip(cache, (NAN, INF))]
    assert torch.equal(clean, impls.attn_paged(q, *(c.to(DEV) for c in dirty), *rest))
    held = [mxfp4_of(c) for c in cache]
    four = impls.attn_paged_mxfp4(q, *(t.to(DEV) for h in held for t in h), *rest)
    for codes, scales in held:
        scales.masked_fill_(~mine[:, None, None], 255)
        codes.masked_fill_(~mine[:, None, :, None], 0x77)
    assert torch.equal(four, impls.attn_paged_mxfp4(q, *(t.to(DEV) for h in held for t in h), *rest))


@pytest.mark.parametrize("dtype", [BF, F16, F32], ids=str)
@pytest.mark.parametrize("where", ["k", "v"])
def test_nonfinite_keys_reach_only_the_tokens_that_see_them(dtype, where):
    """Key 75 of 100 is a NaN (an Inf among the values): of 40 new tokens the first 15 do not see it."""
    n, ps, d = 100, 16, 64
    k, v = cache_of(7, 2, ps, d, dtype, 4)
    table = torch.arange(7, dtype=torch.int32)[None]
    q = torch.randn(40, 4, d, generator=torch.Generator().manual_seed(3)).to(dtype).to(DEV)
    rest = (table.to(DEV), torch.tensor([n], dtype=torch.int32).to(DEV), torch.tensor([0, 40], dtype=torch.int32).to(DEV))
    clean = impls.attn_paged(q, k.to(DEV), v.to(DEV), *rest).cpu()
    held = [mxfp4_of(c) for c in (k, v)]
    four = impls.attn_paged_mxfp4(q, *(t.to(DEV) for h in held for t in h), *rest).cpu()
    (k if where == "k" else v)[75 // ps, 1, 75 % ps, 5] = NAN if where == "k" else INF
    got = impls.attn_paged(q, k.to(DEV), v.to(DEV), *rest).cpu()
    held[0 if where == "k" else 1][1][75 // ps, 1, 0, 75 % ps] = 255
    got4 = impls.attn_paged_mxfp4(q, *(t.to(DEV) for h in held for t in h), *rest).cpu()
    blind = 75 - (n - 40)
    for a, b in ((got, clean), (got4, four)):
        assert torch.equal(a[:, :2], b[:, :2])  # kv head 0
        # a tile is taken key by key where something in it is not finite: another order of the same sum
        torch.testing.assert_close(a[:blind, 2:], b[:blind, 2:], rtol=4 * HALF_STEP[dtype], atol=4 * HALF_STEP[dtype])
    if where == "k":
        assert got[blind:, 2:].isnan().all() and got4[blind:, 2:].isnan().all()
    else:
        assert (got[blind:, 2:, 5] == INF).all() and got[blind:, 2:, :5].isfinite().all()
        assert got4[blind:, 2:, :32].isnan().all() and got4[blind:, 2:, 32:].isfinite().all()


@pytest.mark.parametrize("dtype", [BF, F16, F32], ids=str)
@pytest.mark.parametrize("news", [[1, 1], [20, 3], [300, 3]], ids=str)
def test_infinite_values_are_infinite_results(dtype, news):
    """An Inf among the values of a key that every token sees: P times it is that Inf, in whatever terms P is held."""
    ps, d, lens = 16, 64, [400, 30]
    k, v = cache_of(27, 2, ps, d, dtype, 4)
    table = table_of(lens, ps, 27, 25, 5)
    total = sum(news)
    q = torch.randn(total, 4, d, generator=torch.Generator().manual_seed(3)).to(dtype).mul_(0.25).to(DEV)
    cu = torch.tensor([0, news[0], total], dtype=torch.int32)
    v[table[0, 2], 1, 5, 7], v[table[1, 0], 0, 3, 9] = INF, -INF
    got = impls.attn_paged(q, k.to(DEV), v.to(DEV), table.to(DEV), torch.tensor(lens, dtype=torch.int32).to(DEV), cu.to(DEV)).cpu()
    first, second = got[:news[0]], got[news[0]:]
    assert (first[:, 2:, 7] == INF).all() and (second[:, :2, 9] == -INF).all()
    first[:, 2:, 7], second[:, :2, 9] = 0, 0
    assert got.isfinite().all()


def test_rows_without_a_finite_score():
    """Scores that are all -Inf are 0 / 0, as softmax has it; +Inf among them is a NaN as well."""
    k, v = cache_of(2, 1, 16, 64, F32, 4)
    k[:] = 0
    k[..., 0] = -INF
    q = torch.zeros(2, 1, 64)
    q[:, :, 0] = 1.0
    rest = (torch.tensor([[0, 1], [1, 0]], dtype=torch.int32).to(DEV), torch.tensor([20, 0], dtype=torch.int32).to(DEV))
    got = impls.attn_paged(q.to(DEV), k.to(DEV), v.to(DEV), *rest).cpu()
    assert got[0].isnan().all() and not got[1].any()
    k[0, 0, 3, 0] = INF
    assert impls.attn_paged(q.to(DEV), k.to(DEV), v.to(DEV), *rest).cpu()[0].isnan().all()


@pytest.mark.parametrize("dtype", [BF, F32], ids=str)
def test_growing_scores(dtype):
    """Scores that rise by hundreds along the keys, so the running maximum moves all the way, and that fall."""
    n, ps, d = 600, 16, 64
    for sign in (1.0, -1.0):
        k, v = cache_of(38, 1, ps, d, dtype, 4)
        k[:] = 0
        k[:, 0, :, 0] = (sign * torch.arange(38 * ps).view(38, ps)).to(dtype)
        q = torch.zeros(1, 2, d, dtype=dtype)
        q[:, :, 0] = 8.0
        table, lens = torch.arange(38, dtype=torch.int32)[None], torch.tensor([n], dtype=torch.int32)
        got = impls.attn_paged(q.to(DEV), k.to(DEV), v.to(DEV), table.to(DEV), lens.to(DEV))
        check(got, exact(q, k, v, table, [n], None, True, None), dtype, d, n)


def test_every_scale_byte():
    """E8M0 bytes 0 to 254 in the values' scales stand for 2^(byte - 127), 255 for NaN."""
    ps, d = 256, 32
    codes = torch.randint(0, 256, (1, 1, ps, d // 2), generator=torch.Generator().manual_seed(1)).to(torch.uint8)
    k_scales = torch.full((1, 1, 1, ps), 127, dtype=torch.uint8)
    v_scales = torch.arange(256, dtype=torch.uint8).view(1, 1, 1, ps)
    for dtype in (BF, F32):
        q = torch.zeros(1, 1, d, dtype=dtype)
        for n in (1, 60, 120, 200, 250):  # one key alone, through the first page entry of a table that starts anywhere
            v = v_scales.roll(-n + 1, dims=-1)
            vc = codes.roll(-n + 1, dims=-2)
            got = impls.attn_paged_mxfp4(q.to(DEV), codes.to(DEV), k_scales.to(DEV), vc.to(DEV), v.to(DEV),
                                         torch.zeros(1, 1, dtype=torch.int32).to(DEV), torch.tensor([1], dtype=torch.int32).to(DEV))
            assert torch.equal(got.cpu()[0, 0].double(), values_of(vc, v)[0, 0, 0].to(dtype).double()), (dtype, n)
    got = impls.attn_paged_mxfp4(q.to(DEV), codes.to(DEV), k_scales.to(DEV), codes.to(DEV), v_scales.to(DEV),
                                 torch.zeros(1, 1, dtype=torch.int32).to(DEV), torch.tensor([256], dtype=torch.int32).to(DEV))
    assert got.isnan().all()


@pytest.mark.parametrize("mxfp4", [False, True], ids=["rows", "mxfp4"])
def test_strides(mxfp4):
    """A token-major pool, keys and values interleaved in one buffer, queries inside a packed projection, a wide table."""
    lens, ps, d, hkv = [90, 33, 200], 16, 64, 2
    cache = cache_of(24, hkv, ps, d, BF, 6)
    table = table_of(lens, ps, 24, 13, 7)
    wide = torch.full((3, 40), 10 ** 6, dtype=torch.int32)
    wide[:, 5:18] = table
    qkv = torch.randn(3, 4 + 2 * hkv, d, generator=torch.Generator().manual_seed(8)).to(BF).to(DEV)
    lens_t = torch.tensor(lens, dtype=torch.int32).to(DEV)

    def token_major(t):  # [pages, heads, ps, x] over memory [pages, ps, 2, heads, x]
        pool = torch.zeros(t.shape[0], ps, 2, hkv, t.shape[3], dtype=t.dtype, device=DEV)
        view = pool[:, :, 1].permute(0, 2, 1, 3)
        view.copy_(t)
        return view

    if mxfp4:
        held = [mxfp4_of(c) for c in cache]
        dense = [t.to(DEV) for h in held for t in h]
        loose = [token_major(dense[0]), dense[1][:, :, :, :], token_major(dense[2]), dense[3]]
        op = impls.attn_paged_mxfp4
    else:
        dense = [c.to(DEV) for c in cache]
        loose = [token_major(c) for c in dense]
        op = impls.attn_paged
    want = op(qkv[:, :4].contiguous(), *dense, table.to(DEV), lens_t)
    assert torch.equal(op(qkv[:, :4], *loose, wide.to(DEV)[:, 5:18], lens_t), want)


# ------------------------------------------------------------------ appending


def _append_inputs(tokens, hq, hkv, d, half, dtype, tables, positions, pages, ps, seed=0):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(tokens, hq + 2 * hkv, d, generator=g).to(dtype)
    angle = torch.rand(positions, half, generator=g) * 6.28
    at = torch.randint(0, positions, (tokens,), generator=g)
    slots = torch.randperm(pages * ps, generator=g)[:tokens]
    return qkv, angle.cos().to(tables), angle.sin().to(tables), at, slots


@pytest.mark.parametrize("dtype", [BF, F16, F32], ids=str)
@pytest.mark.parametrize("interleaved", [False, True], ids=["neox", "gptj"])
@pytest.mark.parametrize("shape", [(1, 1, 1, 8, 4), (37, 8, 2, 128, 64), (5, 3, 1, 40, 20), (5, 3, 1, 40, 7), (300, 12, 4, 96, 24),
                                   (17, 2, 2, 256, 128), (64, 5, 5, 72, 36)], ids=str)
def test_rope_append(shape, interleaved, dtype):
    tokens, hq, hkv, d, half = shape
    pages, ps = 25, 16
    for tables in {F32, dtype}:
        qkv, cos, sin, at, slots = _append_inputs(tokens, hq, hkv, d, half, dtype, tables, 50, pages, ps)
        slots[tokens // 2] = -1 if tokens > 1 else slots[0]
        if tokens > 3:
            slots[1] = pages * ps  # behind the pool: not written
        caches = cache_of(pages, hkv, ps, d, dtype, 5)
        want_caches = [c.clone() for c in caches]
        q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        # the reference's roundings are the op's: fp32 products and sum, rounded once
        want = R.rope_append(q, k, v, cos, sin, at, slots, *want_caches, interleaved)
        dev = [c.to(DEV) for c in caches]
        moved = qkv.to(DEV)
        for narrow in (torch.int64, torch.int32):
            got = impls.rope_append(moved[:, :hq], moved[:, hq:hq + hkv], moved[:, hq + hkv:], cos.to(DEV), sin.to(DEV),
                                    at.to(narrow).to(DEV), slots.to(narrow).to(DEV), *dev, interleaved)
            for a, b in zip((*got, *dev), (*want, *want_caches)):
                assert torch.equal(a.cpu(), b), f"{shape} {dtype} {tables}"


@pytest.mark.parametrize("dtype", [BF, F16, F32], ids=str)
@pytest.mark.parametrize("interleaved", [False, True], ids=["neox", "gptj"])
@pytest.mark.parametrize("shape", [(1, 1, 1, 32, 16), (37, 8, 2, 128, 64), (300, 6, 3, 96, 24), (17, 2, 2, 256, 128),
                                   (9, 2, 1, 64, 11), (40, 1, 1, 160, 80)], ids=str)
def test_rope_append_mxfp4(shape, interleaved, dtype):
    """Codes, scales and what they stand for, to the bit."""
    tokens, hq, hkv, d, half = shape
    pages, ps = 25, 16
    for tables in {F32, dtype}:
        qkv, cos, sin, at, slots = _append_inputs(tokens, hq, hkv, d, half, dtype, tables, 50, pages, ps)
        qkv[:, hq + hkv:, :32] *= 2.0 ** -9
        slots[tokens // 2] = -1 if tokens > 1 else slots[0]
        held = [t for c in cache_of(pages, hkv, ps, d, dtype, 5) for t in mxfp4_of(c)]
        want_held = [t.clone() for t in held]
        q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        want = R.rope_append_mxfp4(q, k, v, cos, sin, at, slots, *want_held, interleaved)
        dev = [t.to(DEV) for t in held]
        moved = qkv.to(DEV)
        got = impls.rope_append_mxfp4(moved[:, :hq], moved[:, hq:hq + hkv], moved[:, hq + hkv:], cos.to(DEV), sin.to(DEV),
                                      at.to(DEV), slots.to(DEV), *dev, interleaved)
        for name, a, b in zip(("yq", "yk", "yv", "k_codes", "k_scales", "v_codes", "v_scales"), (*got, *dev),
                              (*want, *want_held)):
            assert torch.equal(a.cpu(), b), f"{name} {shape} {dtype} {tables}"


def test_mxfp4_borders():
    """Ties, saturation, zeros of both signs, the smallest and largest blocks, and blocks that are not finite."""
    grid = [0.0, 0.25, 0.5, 0.75, 1.0, 1.25, 1.5, 1.75, 2.0, 2.5, 3.0, 3.5, 4.0, 5.0, 6.0, 7.0]
    rows = []
    for power in (0, -5, 90, -120, -126, -127, -130, 125):
        for top in (4.0, 6.0, 7.875, 5.0):
            v = torch.tensor(grid + [-x for x in grid]) * 2.0 ** power
            v = torch.where(v.abs() > top * 2.0 ** power, torch.tensor(top * 2.0 ** power), v)
            rows.append(v)
    rows.append(torch.zeros(32))
    for bad in (NAN, INF, -INF):
        v = torch.ones(32)
        v[7] = bad
        rows.append(v)
    v = torch.stack(rows)[:, None]  # [tokens, 1, 32]
    n = v.shape[0]
    cos, sin = torch.ones(4, 16), torch.zeros(4, 16)
    at, slots = torch.zeros(n, dtype=torch.int64), torch.arange(n)
    held = [torch.zeros(4, 1, 16, 16, dtype=torch.uint8), torch.zeros(4, 1, 1, 16, dtype=torch.uint8)]
    held = held + [t.clone() for t in held]
    dev = [t.to(DEV) for t in held]
    # through the values and, turned by nothing, through the keys
    k = torch.where(v.isfinite(), v, 1.0)
    want = R.rope_append_mxfp4(k, k, v, cos, sin, at, slots, *held)
    got = impls.rope_append_mxfp4(k.to(DEV), k.to(DEV), v.to(DEV), cos.to(DEV), sin.to(DEV), at.to(DEV), slots.to(DEV), *dev)
    for name, a, b in zip(("yk", "yv"), got[1:], want[1:]):
        same = (a.cpu() == b) | (a.cpu().isnan() & b.isnan())
        assert same.all(), name
    for name, a, b in zip(("k_codes", "k_scales", "v_codes", "v_scales"), dev, held):
        assert torch.equal(a.cpu(), b), name


def test_append_strides_and_far_rows():
    """A token-major pool and a row whose byte offset passes 32 bits; tokens on their own strides."""
    d, ps, hkv = 128, 16, 1
    pages = (1 << 31) // (ps * d * 2) + 64  # 2 GiB and more of bf16
    k_cache = torch.zeros(pages, ps, hkv, d, dtype=BF, device=DEV).permute(0, 2, 1, 3)
    v_cache = torch.zeros(pages, hkv, ps, d, dtype=BF, device=DEV)
    qkv = torch.randn(3, 4, d, generator=torch.Generator().manual_seed(1)).to(BF).to(DEV)
    cos, sin = torch.rand(9, 64).to(DEV), torch.rand(9, 64).to(DEV)
    slots = torch.tensor([pages * ps - 1, 5, pages * ps - 40], device=DEV)
    yq, yk = impls.rope_append(qkv[:, :2], qkv[:, 2:3], qkv[:, 3:], cos, sin, torch.tensor([0, 8, 100], device=DEV), slots,
                               k_cache, v_cache)
    for t, s in enumerate(slots.tolist()):
        assert torch.equal(k_cache[s // ps, :, s % ps], yk[t]) and torch.equal(v_cache[s // ps, :, s % ps], qkv[t, 3:])
    at = R.rotary_embedding(qkv[2:3, :2].cpu()[None], cos[8:9].cpu(), sin[8:9].cpu())  # position 100: the table's last row
    assert torch.equal(yq[2:3].cpu(), at[0])
    # and attention finds them there
    table = torch.tensor([[pages - 1, 0], [0, 0], [(pages * ps - 40) // ps, 0]], dtype=torch.int32)
    lens = [16, 6, ps - 40 % ps + 1]
    got = impls.attn_paged(yq, k_cache, v_cache, table.to(DEV), torch.tensor(lens, dtype=torch.int32).to(DEV))
    small = [torch.stack([c[p] for p in (pages - 1, 0, (pages * ps - 40) // ps)]).cpu() for c in (k_cache, v_cache)]
    near = torch.tensor([[0, 0], [1, 0], [2, 0]], dtype=torch.int32)
    check(got, exact(yq.cpu(), *small, near, lens, None, True, None), BF, d, 16)


def _far(shape, gap, at, dtype, buf=None):
    """A zeroed view of `shape` [3, heads, a, b] whose pages lie `gap` bytes apart, `at` bytes into a buffer."""
    size = dtype.itemsize
    n = shape[1] * shape[2] * shape[3]
    if buf is None:
        buf = torch.empty((2 * gap + 8 * n * size) // size, dtype=dtype, device=DEV)
    view = buf.as_strided(shape, (gap // size, shape[2] * shape[3], shape[3], 1), at // size)
    return view.zero_(), buf


@pytest.mark.parametrize("news", [None, [40, 33]], ids=str)
@pytest.mark.parametrize("mxfp4", [False, True], ids=["rows", "mxfp4"])
def test_pages_four_gib_apart(mxfp4, news):
    """Offsets past 32 bits, of keys, values and scales, in attention and in appending."""
    hkv, ps, d, gap = 2, 16, 64, (1 << 32) + 4096
    lens, table = [40, 33], torch.tensor([[2, 0, 1], [1, 2, 0]], dtype=torch.int32)
    n = 2 if news is None else sum(news)
    cache = cache_of(3, hkv, ps, d, BF, 5)
    if mxfp4:
        held = [mxfp4_of(c) for c in cache]
        rows = [values_of(*h) for h in held]
        flat = [t for h in held for t in h]
    else:
        rows = flat = list(cache)
    views, buf = [], None
    for t in flat:
        view, buf = _far(tuple(t.shape), gap, sum(2 * v[0].numel() * v.element_size() for v in views), t.dtype, buf)
        views.append(view)
    assert len({v.stride(0) for v in views}) == 1
    for v, t in zip(views, flat):
        v.copy_(t)
    q = torch.randn(n, 8, d, generator=torch.Generator().manual_seed(6)).to(BF)
    cu = None if news is None else torch.tensor([0, news[0], n], dtype=torch.int32)
    op = impls.attn_paged_mxfp4 if mxfp4 else impls.attn_paged
    got = op(q.to(DEV), *views, table.to(DEV), torch.tensor(lens, dtype=torch.int32).to(DEV), None if cu is None else cu.to(DEV))
    check(got, exact(q, *rows, table, lens, cu, True, None), BF, d, 40, mxfp4)
    append = impls.rope_append_mxfp4 if mxfp4 else impls.rope_append
    k, v = (torch.randn(2, hkv, d, generator=torch.Generator().manual_seed(s)).to(BF) for s in (7, 8))
    one, none = torch.ones(1, d // 2), torch.zeros(1, d // 2)
    args = q[:2], k, v, one, none, torch.zeros(2, dtype=torch.int64), torch.tensor([2 * ps + 3, ps + 15])
    want = [t.clone() for t in flat]
    (R.rope_append_mxfp4 if mxfp4 else R.rope_append)(*args, *want)
    append(*(t.to(DEV) for t in args), *views)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(views, want))


def test_rotated_keys_past_the_largest_fp32_are_nan_blocks():
    """x cos + partner sin between the largest fp32 and 2^128, in 64 bits: no fp32 value; one below it is finite."""
    top = torch.finfo(torch.float32).max
    k = torch.zeros(2, 1, 64)
    k[0, 0, 3], k[0, 0, 3 + 32] = top, 2.0 ** 101  # top + 2^101, less than half a step above top
    k[1, 0, 3], k[1, 0, 3 + 32] = top, -(2.0 ** 101)
    cos, sin = torch.ones(1, 32), torch.full((1, 32), -1.0)
    cos[:, :3], cos[:, 4:], sin[:, :3], sin[:, 4:] = 1, 1, 0, 0
    args = k, k, k, cos, sin, torch.zeros(2, dtype=torch.int32), torch.arange(2, dtype=torch.int32)
    outs = []
    for dev, op in (("cpu", R.rope_append_mxfp4), (DEV, impls.rope_append_mxfp4)):
        held = [torch.zeros(1, 1, 16, 32, dtype=torch.uint8), torch.zeros(1, 1, 2, 16, dtype=torch.uint8)]
        held = [t.to(dev) for t in (*held, *(t.clone() for t in held))]
        ys = op(*(t.to(dev) for t in args), *held)
        outs.append([t.cpu() for t in (*ys[1:], *held)])
    assert outs[0][0][0, 0, :32].isnan().all() and outs[0][0][1, 0, :32].isfinite().all()
    assert all(torch.equal(a.nan_to_num(7.0) if a.is_floating_point() else a, b.nan_to_num(7.0) if b.is_floating_point() else b)
               for a, b in zip(*outs))


# ------------------------------------------------------------------ as a program uses them


def test_answering_token_by_token():
    """A prompt appended and attended whole, then single tokens, against attention over the whole sequence at the end;
    with the 4-bit cache the prompt attends yk and yv, which is what the cache holds."""
    hq, hkv, d, ps, prompt, steps = 8, 2, 64, 16, 45, 6
    total = prompt + steps
    g = torch.Generator().manual_seed(4)
    qkv = torch.randn(total, hq + 2 * hkv, d, generator=g).to(BF).to(DEV)
    angle = torch.rand(64, 32, generator=g) * 6.28
    cos, sin = angle.cos().to(DEV), angle.sin().to(DEV)
    table = torch.tensor([[5, 2, 7, 0]], dtype=torch.int32).to(DEV)
    at = torch.arange(total).to(DEV)
    slots = table[0].long()[at // ps] * ps + at % ps
    for mxfp4 in (False, True):
        if mxfp4:
            cache = [torch.zeros(8, hkv, ps, d // 2, dtype=torch.uint8, device=DEV),
                     torch.zeros(8, hkv, d // 32, ps, dtype=torch.uint8, device=DEV)]
            cache = cache + [t.clone() for t in cache]
            append, attend = impls.rope_append_mxfp4, impls.attn_paged_mxfp4
        else:
            cache = [torch.zeros(8, hkv, ps, d, dtype=BF, device=DEV) for _ in range(2)]
            append, attend = impls.rope_append, impls.attn_paged
        outs, ks, vs, qs = [], [], [], []
        for first, last in [(0, prompt), *((i, i + 1) for i in range(prompt, total))]:
            part = qkv[first:last]
            y = append(part[:, :hq], part[:, hq:hq + hkv], part[:, hq + hkv:], cos, sin, at[first:last], slots[first:last],
                       *cache)
            qs.append(y[0])
            ks.append(y[1])
            vs.append(y[2] if mxfp4 else part[:, hq + hkv:])
            cu = torch.tensor([0, last - first], dtype=torch.int32, device=DEV)
            outs.append(attend(y[0], *cache, table, torch.tensor([last], dtype=torch.int32, device=DEV), cu))
        q, k, v = (torch.cat(t) for t in (qs, ks, vs))
        got = torch.cat(outs)
        dense = exact(q.cpu(), k.cpu().transpose(0, 1)[None], v.cpu().transpose(0, 1)[None],
                      torch.zeros(1, 1, dtype=torch.int32), [total], torch.tensor([0, total]), True, None)
        check(got, dense, BF, d, total, mxfp4)
        whole = impls.attn_varlen(q, k, v.contiguous(), torch.tensor([0, total], dtype=torch.int32), True)
        check(whole, dense, BF, d, total, mxfp4)


@pytest.mark.parametrize("mxfp4", [False, True], ids=["rows", "mxfp4"])
def test_captured_steps_replay_with_other_lengths(mxfp4):
    """A decode step (append, then attention) captured once and replayed as its sequences grow, pages are added and
    requests leave (slot -1, length 0), with eager calls between: every replay equals the eager step."""
    hq, hkv, d, ps, seqs, width = 8, 2, 64, 16, 5, 64
    pages = seqs * width
    if mxfp4:
        cache = [t.to(DEV) for c in cache_of(pages, hkv, ps, d, BF, 1) for t in mxfp4_of(c)]
        append, attend = impls.rope_append_mxfp4, impls.attn_paged_mxfp4
    else:
        cache = [c.to(DEV) for c in cache_of(pages, hkv, ps, d, BF, 1)]
        append, attend = impls.rope_append, impls.attn_paged
    cos, sin = torch.rand(1024, 32, device=DEV), torch.rand(1024, 32, device=DEV)
    qkv = torch.zeros(seqs, hq + 2 * hkv, d, dtype=BF, device=DEV)
    at = torch.zeros(seqs, dtype=torch.int64, device=DEV)
    slots = torch.zeros(seqs, dtype=torch.int64, device=DEV)
    lens = torch.ones(seqs, dtype=torch.int32, device=DEV)
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(2)).int().view(seqs, width).to(DEV)

    def step(held):
        y = append(qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:], cos, sin, at, slots, *held)
        return (*y, attend(y[0], *held, table, lens))

    def fill(seed):
        g = torch.Generator().manual_seed(seed)
        n = torch.randint(1, 1000, (seqs,), generator=g)
        n[seed % seqs] = 0
        qkv.copy_(torch.randn(qkv.shape, generator=g))
        at.copy_((n - 1).clamp(min=0))
        row = (n - 1).clamp(min=0).to(DEV)
        slots.copy_(torch.where(n.to(DEV) > 0, table.long().gather(1, (row // ps)[:, None])[:, 0] * ps + row % ps, -1))
        lens.copy_(n)

    fill(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step([t.clone() for t in cache])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(cache)
    for seed in range(1, 5):
        fill(seed)
        before = [t.clone() for t in cache]
        graph.replay()
        torch.cuda.synchronize()
        eager = step(before)
        torch.cuda.synchronize()
        for a, b in zip((*captured, *cache), (*eager, *before)):
            assert torch.equal(a, b)


def test_two_streams_at_once():
    a, b = ([c.to(DEV) for c in cache_of(300, 2, 16, 128, BF, s)] for s in (1, 2))
    table = torch.randperm(300, generator=torch.Generator().manual_seed(3)).int().view(2, 150).to(DEV)
    lens = torch.tensor([2400, 1999], dtype=torch.int32).to(DEV)
    q = torch.randn(2, 16, 128, generator=torch.Generator().manual_seed(4)).to(BF).to(DEV)
    want = [impls.attn_paged(q, *c, table, lens) for c in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        got = []
        for s, c in zip(streams, (a, b)):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(impls.attn_paged(q, *c, table, lens))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_native_and_python_paths_agree(monkeypatch):
    cache = [c.to(DEV) for c in cache_of(20, 2, 16, 64, BF, 1)]
    held = [t.to(DEV) for c in cache_of(20, 2, 16, 64, BF, 1) for t in mxfp4_of(c)]
    table = torch.arange(20, dtype=torch.int32).view(2, 10).to(DEV)
    lens, cu = torch.tensor([150, 77], dtype=torch.int32).to(DEV), torch.tensor([0, 3, 5], dtype=torch.int32).to(DEV)
    qkv = torch.randn(5, 12, 64, generator=torch.Generator().manual_seed(4)).to(BF).to(DEV)
    cos, sin = torch.rand(9, 32, device=DEV), torch.rand(9, 32, device=DEV)
    at, slots = torch.arange(5, device=DEV), torch.arange(5, device=DEV) * 3
    part = qkv[:, :8], qkv[:, 8:10], qkv[:, 10:]

    def calls():
        return (*impls.rope_append(*part, cos, sin, at, slots, *cache), impls.attn_paged(part[0], *cache, table, lens, cu),
                impls.attn_paged(part[0][:2], *cache, table, lens, None, True, 0.5),
                *impls.rope_append_mxfp4(*part, cos, sin, at, slots, *held),
                impls.attn_paged_mxfp4(part[0], *held, table, lens, cu, False), *cache, *held)

    native = _lib.native()
    for name in ("rope_append", "rope_append_mxfp4", "attn_paged", "attn_paged_mxfp4"):
        assert hasattr(native, name)
    assert native.attn_paged(part[0], *cache, table, lens, cu, True, None) is not NotImplemented
    assert native.rope_append_mxfp4(*part, cos, sin, at, slots, *held, False) is not NotImplemented
    first = [t.clone() for t in calls()]
    monkeypatch.setattr(_lib, "_native", _lib._ThroughPython())
    assert all(torch.equal(a, b) for a, b in zip(first, calls()))


def test_refusals():
    cache = [c.to(DEV) for c in cache_of(4, 2, 16, 64, BF, 1)]
    held = [t.to(DEV) for c in cache_of(4, 2, 16, 64, BF, 1) for t in mxfp4_of(c)]
    q = torch.randn(2, 4, 64, device=DEV).to(BF)
    k = torch.randn(2, 2, 64, device=DEV).to(BF)
    table, lens = torch.zeros(2, 2, dtype=torch.int32, device=DEV), torch.ones(2, dtype=torch.int32, device=DEV)
    cos = torch.rand(9, 32, device=DEV)
    at = torch.arange(2, device=DEV)
    with pytest.raises(RuntimeError, match="no gradient"):
        impls.attn_paged(q.clone().requires_grad_(), *cache, table, lens)
    with pytest.raises(RuntimeError, match="no gradient"):
        impls.rope_append(q, k.clone().requires_grad_(), k, cos, cos, at, at, *cache)
    with pytest.raises(TypeError, match="int32"):
        impls.attn_paged(q, *cache, table.long(), lens)
    with pytest.raises(TypeError, match="cache of"):
        impls.attn_paged(q.half(), *cache, table, lens)
    with pytest.raises(ValueError, match="multiple of kv_heads"):
        impls.attn_paged(q[:, :3], *cache, table, lens)
    with pytest.raises(ValueError, match="cache_lens"):
        impls.attn_paged(q, *cache, table, lens[:1])
    with pytest.raises(ValueError, match="page_size"):
        impls.attn_paged(q, *(c[:, :, :8] for c in cache), table, lens)
    with pytest.raises(ValueError, match="contiguous"):
        impls.attn_paged(q[..., :32], *(c[..., ::2] for c in cache), table, lens)
    with pytest.raises(_lib.KernelError, match="16-byte aligned|multiple of 16 bytes"):
        impls.attn_paged(q[..., :56], *(c[..., 1:57] for c in cache), table, lens)
    with pytest.raises(ValueError, match="share memory"):
        impls.rope_append(q, k, k, cos, cos, at, at, *(c[:1].expand(4, -1, -1, -1) for c in cache))
    with pytest.raises(ValueError, match="slots"):
        impls.rope_append(q, k, k, cos, cos, at, at.float(), *cache)
    with pytest.raises(ValueError, match="cos/sin"):
        impls.rope_append(q, k, k, torch.rand(9, 33, device=DEV), torch.rand(9, 33, device=DEV), at, at, *cache)
    with pytest.raises(TypeError, match="uint8"):
        impls.attn_paged_mxfp4(q, held[0].to(torch.int8), *held[1:], table, lens)
    with pytest.raises(ValueError, match="scales"):
        impls.attn_paged_mxfp4(q, held[0], held[1][..., :8], *held[2:], table, lens)
    # nothing to do
    assert impls.attn_paged(q[:0], *cache, table[:0], lens[:0]).shape == (0, 4, 64)
    none = impls.attn_paged(q, *cache, table[:0], lens[:0], torch.zeros(1, dtype=torch.int32, device=DEV))
    assert not none.any()
    yq, yk = impls.rope_append(q[:0], k[:0], k[:0], cos, cos, at[:0], at[:0], *cache)
    assert yq.shape == (0, 4, 64) and yk.shape == (0, 2, 64)


def test_caches_of_different_strides_are_refused():
    cache = [c.to(DEV) for c in cache_of(4, 2, 16, 64, BF, 1)]
    held = [t.to(DEV) for c in cache_of(4, 2, 16, 64, BF, 1) for t in mxfp4_of(c)]
    q = torch.randn(2, 4, 64, device=DEV).to(BF)
    table, lens = torch.zeros(2, 2, dtype=torch.int32, device=DEV), torch.ones(2, dtype=torch.int32, device=DEV)
    other = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in held]
    with pytest.raises(_lib.KernelError, match="different strides"):
        impls.attn_paged(q, cache[0], cache[1].transpose(1, 2).contiguous().transpose(1, 2), table, lens)
    with pytest.raises(_lib.KernelError, match="codes|key and the value"):
        impls.attn_paged_mxfp4(q, held[0], held[1], other[2], held[3], table, lens)
    with pytest.raises(_lib.KernelError, match="scales have different strides"):
        impls.attn_paged_mxfp4(q, held[0], held[1], held[2], other[3], table, lens)
    assert torch.equal(impls.attn_paged(q, *cache, table, lens), impls.attn_paged(q, *cache, table, lens))


def test_records_and_routes(monkeypatch, tmp_path):
    """Through the dispatch: each op graded against its reference by the harness, and then served by the backend."""
    from popcorn_amd import backend, compat
    from popcorn_amd.compat import store

    monkeypatch.setattr(store, "BUNDLED_REPORTS", tmp_path / "bundled")
    backend.register(compat)
    g = torch.Generator().manual_seed(0)
    tokens, hq, hkv, d, ps, pages = 24, 8, 2, 64, 16, 12
    q, k, v = (torch.randn(tokens, h, d, generator=g).to(BF).to(DEV) for h in (hq, hkv, hkv))
    angle = torch.rand(64, d // 2, generator=g) * 6.28
    cos, sin = angle.cos().to(BF).to(DEV), angle.sin().to(BF).to(DEV)  # one float type, as a recorded call has
    at, slots = torch.arange(tokens, device=DEV), torch.randperm(pages * ps, generator=g)[:tokens].to(DEV)
    cache = [c.to(DEV) for c in cache_of(pages, hkv, ps, d, BF, 1)]
    held = [t.to(DEV) for c in cache_of(pages, hkv, ps, d, BF, 1) for t in mxfp4_of(c)]
    table = torch.randperm(pages, generator=g).int().view(3, 4).to(DEV)
    lens = torch.tensor([60, 33, 17], dtype=torch.int32, device=DEV)
    cu = torch.tensor([0, 10, 11, tokens], dtype=torch.int32, device=DEV)
    calls = {"rope_append": (q, k, v, cos, sin, at, slots, *cache), "rope_append_mxfp4": (q, k, v, cos, sin, at, slots, *held),
             "attn_paged": (q, *cache, table, lens, cu), "attn_paged_mxfp4": (q, *held, table, lens, cu)}
    for name, args in calls.items():
        op = compat.KERNELS[name]
        op.tuner.forget()
        with torch.no_grad():
            [record] = op.benchmark(*args, backend=backend.BACKEND)
            assert record.result.status == "pass", (name, record.result.status, record.result.reason)
            assert not record.result.grad and record.result.benchmarked
            op(*args)
        assert op.tuner.last_choice() == backend.BACKEND, name
        op.tuner.forget()
    with torch.no_grad():  # single tokens and fp32 tables: no one config to record, served in registration order
        for name, args in (("attn_paged", (q[:3], *cache, table, lens)), ("attn_paged_mxfp4", (q[:3], *held, table, lens)),
                           ("rope_append", (q, k, v, cos.float(), sin.float(), at, slots, *cache))):
            compat.KERNELS[name](*args)
            assert compat.KERNELS[name].tuner.last_choice() == backend.BACKEND, name
            compat.KERNELS[name].tuner.forget()
