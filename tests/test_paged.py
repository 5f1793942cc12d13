"""The paged cache's ops without a GPU: their references against facts of their own, predicates, refusals, the C entry points."""

from __future__ import annotations

import ctypes
import itertools

import pytest
import torch

from popcorn_amd import _lib, backend, compat, impls
from popcorn_amd.compat import references as R
from popcorn_amd.compat.ops import describe
from tests._paged import cache_of, check, exact, mxfp4_of, table_of, values_of

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ------------------------------------------------------------------ the 4-bit format


def test_mxfp4_takes_the_nearest_value_and_even_codes_on_ties():
    """Against a search of all sixteen values. The scale of a block whose largest magnitude is 4 to 7.9 is 1."""
    points = sorted({m + e for m in (*GRID, *((a + b) / 2 for a, b in zip(GRID, GRID[1:])), 7.9) for e in (-1e-9, 0.0, 1e-9)
                     if 0 <= m + e})
    for chunk in itertools.batched(points, 30) if hasattr(itertools, "batched") else (points[i:i + 30] for i in
                                                                                      range(0, len(points), 30)):
        block = torch.tensor([4.0, -4.0, *chunk], dtype=torch.float64)
        block = torch.cat([block, torch.zeros(32 - block.numel(), dtype=torch.float64)])
        block[2::2] *= -1
        codes, scales = R.mxfp4_encode(block)
        assert scales.tolist() == [127]
        nibbles = [c for byte in codes.tolist() for c in (byte & 15, byte >> 4)]
        for y, code in zip(block.tolist(), nibbles):
            best = min(abs(abs(y) - g) for g in GRID)
            near = [i for i, g in enumerate(GRID) if abs(abs(y) - g) == best]
            want = near[0] if len(near) == 1 else next(i for i in near if i % 2 == 0)
            assert code & 7 == want, (y, code)
            if y:
                assert (code >= 8) == (y < 0)


@pytest.mark.parametrize("power", [-149, -130, -127, -126, -125, -124, -1, 0, 1, 100, 127])
def test_mxfp4_scales_follow_the_largest_magnitude(power):
    block = torch.zeros(32, dtype=torch.float64)
    block[7] = 1.5 * 2.0 ** power if power < 127 else 2.0 ** 127
    codes, scales = R.mxfp4_encode(block)
    assert scales.item() == max(power - 2, -126) + 127
    back = R.mxfp4_decode(codes, scales)
    assert (back[:7] == 0).all() and (back[8:] == 0).all()
    if power >= -124:
        assert back[7] == block[7]  # 4 or 6 scales
    else:
        assert abs(back[7] - block[7]) <= 2.0 ** -126 / 4  # half of the smallest step


def test_mxfp4_blocks_without_a_value():
    codes, scales = R.mxfp4_encode(torch.zeros(64))
    assert codes.sum() == 0 and scales.tolist() == [1, 1]
    for bad in (float("nan"), float("inf"), -float("inf"), 2.0 ** 128):
        y = torch.ones(64, dtype=torch.float64)
        y[40] = bad
        codes, scales = R.mxfp4_encode(y)
        assert scales.tolist() == [125, 255]
        back = R.mxfp4_decode(codes, scales)
        assert (back[:32] == 1).all() and back[32:].isnan().all()
    every = R.mxfp4_decode(torch.full((256, 16), 0x21, dtype=torch.uint8), torch.arange(256, dtype=torch.uint8)[:, None])
    assert every[255].isnan().all()
    for e in (0, 1, 127, 254):
        assert every[e, 0] == 0.5 * 2.0 ** (e - 127) and every[e, 1] == 2.0 ** (e - 127)


# ------------------------------------------------------------------ the references


def _append_inputs(tokens, hq, hkv, d, half, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(tokens, hq, d, generator=g).to(dtype)
    k, v = (torch.randn(tokens, hkv, d, generator=g).to(dtype) for _ in range(2))
    angle = torch.rand(11, half, generator=g) * 6.28
    return q, k, v, angle.cos(), angle.sin(), torch.randint(-2, 14, (tokens,), generator=g)


@pytest.mark.parametrize("interleaved", [False, True], ids=["neox", "gptj"])
def test_append_rotates_and_writes_the_rows_of_its_slots(interleaved):
    q, k, v, cos, sin, at = _append_inputs(5, 3, 2, 32, 12, F32)
    slots = torch.tensor([17, -1, 0, 48, 31])  # 48: behind the pool's three pages
    caches = [torch.full((3, 2, 16, 32), 7.0) for _ in range(2)]
    yq, yk = R.rope_append(q, k, v, cos, sin, at, slots, *caches, interleaved)
    for t in range(5):
        pos = min(max(int(at[t]), 0), 10)
        for x, y in ((q, yq), (k, yk)):
            for j in range(12):
                a, b = (2 * j, 2 * j + 1) if interleaved else (j, j + 12)
                c, s = cos[pos, j], sin[pos, j]
                torch.testing.assert_close(y[t, :, a], x[t, :, a] * c - x[t, :, b] * s, rtol=0, atol=2e-6)
                torch.testing.assert_close(y[t, :, b], x[t, :, b] * c + x[t, :, a] * s, rtol=0, atol=2e-6)
            assert torch.equal(y[t, :, 24:], x[t, :, 24:])
    written = {17: 0, 0: 2, 31: 4}
    for s in range(48):
        for cache, y in zip(caches, (yk, v)):
            row = cache[s // 16, :, s % 16]
            assert torch.equal(row, y[written[s]]) if s in written else (row == 7).all()


def test_append_into_four_bits_returns_what_the_cache_holds():
    q, k, v, cos, sin, at = _append_inputs(6, 2, 2, 64, 32, BF)
    rows = [torch.zeros(2, 2, 16, 32, dtype=torch.uint8) for _ in range(2)]
    scales = [torch.zeros(2, 2, 2, 16, dtype=torch.uint8) for _ in range(2)]
    slots = torch.tensor([3, 30, 9, 16, -5, 15])
    yq, yk, yv = R.rope_append_mxfp4(q, k, v, cos, sin, at, slots, rows[0], scales[0], rows[1], scales[1])
    assert torch.equal(yq, R.rope_append(q, k, v, cos, sin, at, slots, *cache_of(2, 2, 16, 64, BF, 0))[0])
    for y, c, s in zip((yk, yv), rows, scales):
        held = values_of(c, s)
        for t, slot in enumerate(slots.tolist()):
            if slot >= 0:
                assert torch.equal(held[slot // 16, :, slot % 16].to(BF), y[t])
    worst = ((yv.double() - v.double()).abs() / v.double().unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True)
             .expand(-1, -1, -1, 32).flatten(-2))
    assert worst.max() <= 1 / 4 + 2.0 ** -8  # a block's top is below 8 scales, its last value 6: at worst 2 of 8


@pytest.mark.parametrize("mxfp4", [False, True], ids=["rows", "mxfp4"])
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
@pytest.mark.parametrize("dtype", [BF, F16, F32], ids=str)
def test_reference_against_dense_attention(dtype, causal, mxfp4):
    """Pages in any order, one outside the pool, a length of none and a run of none; a sequence without any key is zeros."""
    lens, news, ps, d = [37, 0, 20, 70, 9], [3, 2, 0, 5, 1], 16, 32
    cache = cache_of(14, 2, ps, d, dtype, 1)
    table = table_of(lens, ps, 14, 5, 2)
    table[3, 1] = 14
    cu = torch.tensor([0, 3, 5, 5, 10, 11], dtype=torch.int32)
    q = torch.randn(11, 6, d, generator=torch.Generator().manual_seed(3)).to(dtype)
    lens_t = torch.tensor(lens, dtype=torch.int32)
    if mxfp4:
        held = [mxfp4_of(c) for c in cache]
        rows = [values_of(*h) for h in held]
        got = R.attn_paged_mxfp4(q, *(t for h in held for t in h), table, lens_t, cu, causal, 0.3)
    else:
        rows = cache
        got = R.attn_paged(q, *cache, table, lens_t, cu, causal, 0.3)
    assert not got[3:5].any()
    check(got, exact(q, *rows, table, lens, cu, causal, 0.3), dtype, d, max(lens), mxfp4)


def test_a_sequence_in_pages_is_attn_varlen():
    cu = torch.tensor([0, 21, 34], dtype=torch.int32)
    q = torch.randn(34, 4, 16, generator=torch.Generator().manual_seed(1))
    k, v = (torch.randn(34, 2, 16, generator=torch.Generator().manual_seed(s)) for s in (2, 3))
    caches = [torch.zeros(4, 2, 16, 16) for _ in range(2)]
    table = torch.tensor([[2, 0], [3, 1]], dtype=torch.int32)
    for i in range(2):
        for t in range(int(cu[i]), int(cu[i + 1])):
            j = t - int(cu[i])
            for c, x in zip(caches, (k, v)):
                c[table[i, j // 16], :, j % 16] = x[t]
    got = R.attn_paged(q, *caches, table, torch.tensor([21, 13], dtype=torch.int32), cu)
    torch.testing.assert_close(got, R.attn_varlen(q, k, v, cu, True, None), rtol=0, atol=1e-6)


# ------------------------------------------------------------------ the backend's registration


def _meta(*shape, dtype=BF):
    return torch.empty(shape, dtype=dtype, device="meta")


def _append_args(dtype=BF, d=64, ps=16, table=F32, index=torch.int64):
    return [_meta(3, 4, d, dtype=dtype), _meta(3, 2, d, dtype=dtype), _meta(3, 2, d, dtype=dtype),
            _meta(9, d // 2, dtype=table), _meta(9, d // 2, dtype=table), _meta(3, dtype=index), _meta(3, dtype=index),
            _meta(5, 2, ps, d, dtype=dtype), _meta(5, 2, ps, d, dtype=dtype), False]


def _append4_args(dtype=BF, d=64, ps=16):
    rows = [_meta(5, 2, ps, d // 2, dtype=torch.uint8), _meta(5, 2, d // 32, ps, dtype=torch.uint8)]
    return [*_append_args(dtype, d, ps)[:7], *rows, *rows, False]


def _paged_args(dtype=BF, d=64, ps=16, seqs=3, packed=False):
    return [_meta(3, 4, d, dtype=dtype), _meta(5, 2, ps, d, dtype=dtype), _meta(5, 2, ps, d, dtype=dtype),
            _meta(seqs, 7, dtype=torch.int32), _meta(seqs, dtype=torch.int32),
            _meta(seqs + 1, dtype=torch.int32) if packed else None, True, None]


def _paged4_args(dtype=BF, d=64, ps=16):
    rows = [_meta(5, 2, ps, d // 2, dtype=torch.uint8), _meta(5, 2, d // 32, ps, dtype=torch.uint8)]
    return [_meta(3, 4, d, dtype=dtype), *rows, *rows, *_paged_args(d=d)[3:]]


OPS = {"rope_append": (_append_args, backend.rope_append_supported),
       "rope_append_mxfp4": (_append4_args, backend.rope_append_mxfp4_supported),
       "attn_paged": (_paged_args, backend.attn_paged_supported),
       "attn_paged_mxfp4": (_paged4_args, backend.attn_paged_mxfp4_supported)}


@pytest.mark.parametrize("name", OPS)
def test_predicates(name, monkeypatch):
    monkeypatch.setattr(backend, "_on_hip", lambda *tensors: True)
    args, supported = OPS[name]
    for dtype in (BF, F16, F32):
        assert supported(*args(dtype))
    assert not supported(*args(torch.float64))
    four = "mxfp4" in name
    assert supported(*args(d=96)) and supported(*args(d=256)) and supported(*args(ps=48))
    for d in (288, 48 if four else 36):
        assert not supported(*args(d=d)), d
    for ps in (8, 24):
        assert not supported(*args(ps=ps)), ps

    def but(i, t):
        a = args()
        a[i] = t
        return supported(*a)

    assert not but(0, _meta(3, 5, 64) if "attn" in name else _meta(4, 4, 64))
    if "append" in name:
        assert but(5, _meta(3, dtype=torch.int32)) and not but(6, _meta(3, dtype=F32)) and not but(6, _meta(2, dtype=torch.int64))
        assert not but(3, _meta(9, 33, dtype=F32)) and not but(1, _meta(3, 2, 64, dtype=F16))
        assert not but(7, _meta(1, 2, 16, 32 if four else 64, dtype=torch.uint8 if four else BF).expand(5, -1, -1, -1))
        a = args()
        a[3] = a[4] = _meta(9, 32, dtype=BF)  # tables of another float type
        assert supported(*a)
    else:
        at = 5 if four else 3
        assert not but(at, _meta(3, 7, dtype=torch.int64)) and not but(at, _meta(2, 7, dtype=torch.int32))
        assert not but(at + 1, _meta(4, dtype=torch.int32))
        assert supported(*(args()[:at] + [_meta(2, 7, dtype=torch.int32), _meta(2, dtype=torch.int32),
                                          _meta(3, dtype=torch.int32), False, 0.5]))
        # keys and values (and their scales) a different way apart
        other = _meta(5, 16, 2, 32, dtype=torch.uint8).permute(0, 2, 1, 3) if four else _meta(5, 16, 2, 64).permute(0, 2, 1, 3)
        assert not but(1, other)
        if four:
            assert not but(2, _meta(5, 2, 2, 32, dtype=torch.uint8)[..., :16])
            assert not but(0, _meta(3, 4, 64, dtype=torch.float64))
    if four:
        assert not but(7 if "append" in name else 1, _meta(5, 2, 16, 32, dtype=torch.int8))
        assert not but(8 if "append" in name else 2, _meta(5, 2, 1, 16, dtype=torch.uint8))
    else:
        assert not but(7 if "append" in name else 1, _meta(5, 2, 16, 64, dtype=F16))
        assert not but(7 if "append" in name else 1, _meta(5, 2, 16, 128)[..., ::2])


def test_registered_as_forward_only_and_cpu_calls_served_by_torch():
    backend.register(compat)
    q, k, v, cos, sin, at = _append_inputs(4, 4, 2, 32, 16, F32)
    caches = cache_of(3, 2, 16, 32, F32, 1)
    slots, table = torch.tensor([0, 1, 2, 3]), torch.tensor([[0]], dtype=torch.int32)
    args = (q, k, v, cos, sin, at, slots, *caches)
    op = compat.KERNELS["rope_append"]
    assert op[backend.BACKEND].forward_only and op[backend.BACKEND].refusal(describe(op, args, {}))
    yq, yk = op(*args)
    attend = compat.KERNELS["attn_paged"]
    assert attend[backend.BACKEND].forward_only
    lens, cu = torch.tensor([4], dtype=torch.int32), torch.tensor([0, 4], dtype=torch.int32)
    o = attend(yq, *caches, table, lens, cu)
    torch.testing.assert_close(o, R.attn_varlen(yq, yk, v, cu, True, None), rtol=0, atol=1e-6)
    for name in ("rope_append_mxfp4", "attn_paged_mxfp4"):
        assert compat.KERNELS[name][backend.BACKEND].forward_only


@pytest.mark.parametrize("name", OPS)
def test_generated_inputs_run_the_reference(name):
    """The harness's own inputs of each op: its distinct slots, page numbers, lengths and offsets fit the op."""
    sizes = {"tokens": 6, "q_heads": 4, "kv_heads": 2, "head_dim": 32, "max_positions": 8, "half": 16, "pages": 3,
             "page_size": 16, "packed": 16, "blocks": 1, "total": 6, "sequences": 2, "table_pages": 2, "boundaries": 3}
    g = torch.Generator().manual_seed(0)
    slots = R.distinct_slots(torch.empty(6), sizes, g)
    assert slots[-1] == -1 and slots[:-1].unique().numel() == 5 and int(slots.max()) < 48
    with pytest.raises(ValueError, match="do not fit"):
        R.distinct_slots(torch.empty(49), sizes, g)
    lens, table = R.cached_lengths(torch.empty(2), sizes, g), R.table_entries(torch.empty(2, 2), sizes, g)
    assert lens.dtype == table.dtype == torch.int32 and 1 <= int(lens.min()) and int(lens.max()) <= 32
    assert 0 <= int(table.min()) and int(table.max()) < 3


@pytest.mark.parametrize("call", ["rope_append", "rope_append_mxfp4", "attn_paged", "attn_paged_mxfp4"])
def test_cpu_tensors_are_refused_by_the_kernels_functions(call):
    q, k, v, cos, sin, at = _append_inputs(2, 4, 2, 32, 16, F32)
    caches = cache_of(3, 2, 16, 32, F32, 1)
    held = [t for c in caches for t in mxfp4_of(c)]
    table, lens = torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    args = {"rope_append": (q, k, v, cos, sin, at, at, *caches), "rope_append_mxfp4": (q, k, v, cos, sin, at, at, *held),
            "attn_paged": (q, *caches, table, lens), "attn_paged_mxfp4": (q, *held, table, lens)}[call]
    with pytest.raises(Exception, match="(?i)cuda|hip|device"):
        getattr(impls, call)(*args)


# ------------------------------------------------------------------ the C entry points


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIBRARY.exists():
        pytest.fail(f"{_lib.LIBRARY} is not built; run __graft_entry__.build()")
    return _lib.load()


def _strides(*s):
    return (ctypes.c_int64 * len(s))(*s)


FAKE = ctypes.c_void_p(4096)
ODD = ctypes.c_void_p(4104)  # 8-byte aligned


def _paged_call(lib, mxfp4=False, q=FAKE, cache=FAKE, scales=FAKE, table=FAKE, lens=FAKE, cu=None, o=FAKE, ws=None, ws_bytes=0,
                strides=None, seqs=2, total=2, hq=4, hkv=2, d=64, pages=5, ps=16, width=2, scale=0.125, dtype=_lib.BF16):
    row = d // 2 if mxfp4 else d
    base = [4 * d, d, 2 * ps * row, ps * row, row, 2 * ps * row, ps * row, row]
    if mxfp4:
        base += [2 * d // 32 * ps, d // 32 * ps, ps] * 2
    for i, s in (strides or {}).items():
        base[i] = s
    caches = [cache, scales, cache, scales] if mxfp4 else [cache, cache]
    f = lib.pk_attn_paged_mxfp4 if mxfp4 else lib.pk_attn_paged
    rc = f(q, *caches, table, lens, cu, o, ws, ws_bytes, _strides(*base), seqs, total, hq, hkv, d, pages, ps, width, width,
           scale, 1, dtype, None)
    return rc, lib.pk_last_error().decode()


INVALID, UNSUPPORTED = _lib.ERR_INVALID, _lib.ERR_UNSUPPORTED
REFUSED = [  # what differs from a good call, the status, what the message says
    (dict(total=-1), INVALID, "negative"), (dict(pages=-1), INVALID, "negative"), (dict(width=-1), INVALID, "negative"),
    (dict(dtype=7), UNSUPPORTED, "dtype"), (dict(d=36), UNSUPPORTED, "head_dim"), (dict(d=0), UNSUPPORTED, "head_dim"),
    (dict(d=288), UNSUPPORTED, "head_dim"), (dict(ps=8), UNSUPPORTED, "page_size"), (dict(ps=24), UNSUPPORTED, "page_size"),
    (dict(ps=1 << 21), UNSUPPORTED, "page_size"), (dict(scale=float("nan")), INVALID, "softmax_scale"),
    (dict(scale=float("inf")), INVALID, "softmax_scale"), (dict(hq=3), INVALID, "kv_heads"), (dict(hkv=0), INVALID, "kv_heads"),
    (dict(seqs=3), INVALID, "one token"), (dict(q=None), INVALID, "null"), (dict(o=None), INVALID, "null"),
    (dict(cache=None), INVALID, "null"), (dict(lens=None), INVALID, "null"), (dict(table=None), INVALID, "null"),
    (dict(q=ODD), INVALID, "aligned"), (dict(cache=ODD), INVALID, "aligned"), (dict(strides={0: 252}), INVALID, "stride 0"),
    (dict(strides={1: -64}), INVALID, "stride 1"), (dict(strides={3: 1028, 6: 1028}), INVALID, "stride 3"),
    (dict(strides={2: 4096}), UNSUPPORTED, "different strides"), (dict(strides={7: 128}), UNSUPPORTED, "different strides"),
    (dict(strides={4: 1 << 28, 7: 1 << 28}), UNSUPPORTED, "2 GiB"), (dict(width=1 << 27), UNSUPPORTED, "too large"),
    (dict(total=1 << 30, seqs=1, cu=FAKE), UNSUPPORTED, "too large"), (dict(width=400), INVALID, "workspace"),
    (dict(width=400, ws=FAKE, ws_bytes=100), INVALID, "workspace"),
    (dict(width=400, ws=ODD, ws_bytes=1 << 30), INVALID, "workspace"),
]


@pytest.mark.parametrize("mxfp4", [False, True], ids=["rows", "mxfp4"])
@pytest.mark.parametrize("what,status,said", REFUSED, ids=[str(r[0]) for r in REFUSED])
def test_paged_attention_refuses(lib, mxfp4, what, status, said):
    rc, message = _paged_call(lib, mxfp4, **what)
    assert rc == status and said in message and message.startswith("pk_attn_paged"), (rc, message)


def test_scales_are_checked(lib):
    assert _paged_call(lib, True, scales=None)[0] == INVALID
    rc, message = _paged_call(lib, True, scales=ctypes.c_void_p(4098))
    assert rc == INVALID and "scales" in message
    rc, message = _paged_call(lib, True, strides={8: 66, 11: 66})
    assert rc == INVALID and "stride 8" in message
    rc, message = _paged_call(lib, True, strides={9: 64})
    assert rc == UNSUPPORTED and "scales have different strides" in message
    rc, message = _paged_call(lib, True, strides={10: 1 << 29, 13: 1 << 29})
    assert rc == UNSUPPORTED and "2 GiB" in message


def test_empty_calls_launch_nothing(lib):
    for four in (False, True):
        assert _paged_call(lib, four, total=0, seqs=0, q=None, o=None, cache=None, lens=None, table=None)[0] == _lib.OK
        assert _paged_call(lib, four, hq=0)[0] == _lib.OK
    s = _strides(*[64] * 18)
    assert lib.pk_rope_append(*[None] * 11, s, 0, 4, 2, 64, 32, 9, 5, 16, _lib.BF16, _lib.F32, 1, 1, 0, None) == _lib.OK
    assert lib.pk_rope_append_mxfp4(*[None] * 14, s, 0, 4, 2, 64, 32, 9, 5, 16, _lib.BF16, _lib.F32, 1, 1, 0, None) == _lib.OK


@pytest.mark.parametrize("mxfp4", [False, True], ids=["rows", "mxfp4"])
@pytest.mark.parametrize("what,status,said", [
    (dict(tokens=-1), INVALID, "negative"), (dict(dtype=5), UNSUPPORTED, "dtype"), (dict(cs_dtype=5), UNSUPPORTED, "dtype"),
    (dict(head_dim=36), UNSUPPORTED, "head_dim"), (dict(head_dim=288), UNSUPPORTED, "head_dim"), (dict(half=33), INVALID, "half"),
    (dict(half=0), INVALID, "half"), (dict(rows=0), INVALID, "tables"), (dict(ps=20), UNSUPPORTED, "page_size"),
    (dict(pages=1 << 31), UNSUPPORTED, "too large"), (dict(pointer=None), INVALID, "null"),
], ids=lambda w: str(w) if isinstance(w, dict) else "")
def test_append_refuses(lib, mxfp4, what, status, said):
    a = dict(tokens=3, hq=4, hkv=2, head_dim=64, half=32, rows=9, pages=5, ps=16, dtype=_lib.BF16, cs_dtype=_lib.F32,
             pointer=FAKE)
    a.update(what)
    f = lib.pk_rope_append_mxfp4 if mxfp4 else lib.pk_rope_append
    rc = f(*[a.pop("pointer")] * (14 if mxfp4 else 11), _strides(*[64] * 18), *a.values(), 1, 1, 0, None)
    message = lib.pk_last_error().decode()
    assert rc == status and said in message, (rc, message)


def test_append_checks_the_codes_alignment(lib):
    args = [3, 4, 2, 64, 32, 9, 5, 16, _lib.BF16, _lib.F32, 1, 1, 0, None]
    assert lib.pk_rope_append_mxfp4(*[FAKE] * 14, _strides(*[62] * 18), *args) == INVALID
    assert "multiple of 4" in lib.pk_last_error().decode()
    pointers = [FAKE] * 14
    pointers[10] = ctypes.c_void_p(4098)
    assert lib.pk_rope_append_mxfp4(*pointers, _strides(*[64] * 18), *args) == INVALID
    assert "4-byte aligned" in lib.pk_last_error().decode()


def test_workspace_queries(lib):
    ask = lib.pk_attn_paged_workspace
    for mxfp4 in (0, 1):
        for dtype in (_lib.F32, _lib.BF16, _lib.F16):
            assert ask(0, 0, 0, 32, 8, 128, 4096, dtype, mxfp4) == 0
            assert ask(4, 4, 0, 32, 8, 128, 512, dtype, mxfp4) == 0  # one chunk at most
            assert ask(4, 4, 0, 32, 8, 128, 4096, dtype, mxfp4) > 0
            # a grid that fills the device without splitting: 262144 rows x 8 heads in tiles of 128
            if not (mxfp4 and dtype == _lib.F32):  # 16 rows a tile
                assert ask(4, 65536, 1, 32, 8, 128, 131072, dtype, mxfp4) == 0
            for bad in ((-1, 4, 0, 32, 8, 128, 64), (4, 4, 0, 30, 8, 128, 64), (4, 4, 0, 32, 0, 128, 64),
                        (4, 1 << 30, 1, 32, 8, 128, 64), (4, 4, 0, 32, 8, 128, -1)):
                assert ask(*bad, dtype, mxfp4) == -1, bad
    # partial sums of a block: at most min(4 chunks a sequence, rows + a third of a share each) x 8 heads x 4 rows x 128 fp32,
    # their maxima and sums, and the row tiles' numbers, each to 256 bytes
    items = 4 * 8
    assert ask(4, 4, 0, 32, 8, 128, 4096, _lib.BF16, 0) == items * 8 * 4 * 128 * 4 + items * 8 * 4 * 8 + 256
