"""CPU-only checks of the page pool's boundary: tables, argument structs and the refusals made before any launch."""

import math

import pytest
import torch


def test_rotary_tables_frequencies():
    from shadow_infer_b200.shadowkv import rotary_tables
    cos, sin = rotary_tables(8, 50, device="cpu")
    assert cos.shape == sin.shape == (50, 4) and cos.dtype == torch.float32
    for p in (0, 1, 49):
        for i in range(4):
            angle = p * 10000.0 ** (-i / 4)
            assert abs(float(cos[p, i]) - math.cos(angle)) < 2 ** -24 and abs(float(sin[p, i]) - math.sin(angle)) < 2 ** -24
    assert torch.equal(rotary_tables(8, 50, scaling="linear", factor=2.0, device="cpu")[0][::2], cos[:25])


def test_rotary_tables_scaling():
    from shadow_infer_b200.shadowkv import rotary_tables
    n, rot, factor = 2, 64, 8.0
    plain = torch.atan2(*rotary_tables(rot, n, device="cpu")[::-1])[1]      # the angles of position 1
    ntk = torch.atan2(*rotary_tables(rot, n, scaling="ntk", factor=factor, device="cpu")[::-1])[1]
    assert abs(float(ntk[0] - plain[0])) < 1e-6 and abs(float(ntk[-1] * factor / plain[-1]) - 1) < 1e-5
    cos, sin = rotary_tables(rot, n, scaling="ntk_parts", factor=factor, original_positions=4096, device="cpu")
    parts = torch.atan2(sin, cos)[1]
    turns = 4096 * plain / (2 * math.pi)
    fast, slow = turns > 32, turns < 1
    assert fast.any() and slow.any() and (~fast & ~slow).any()
    assert torch.allclose(parts[fast], plain[fast], rtol=1e-5) and torch.allclose(parts[slow], plain[slow] / factor, rtol=1e-5)
    gain = (cos.double() ** 2 + sin.double() ** 2).sqrt()
    assert torch.allclose(gain, torch.full_like(gain, 0.1 * math.log(factor) + 1), rtol=1e-6)


@pytest.mark.parametrize("args,kw", [((7, 4), {}), ((0, 4), {}), ((8, 0), {}), ((8, 4), dict(scaling="spiral")),
                                     ((8, 4), dict(scaling="linear", factor=0.0)), ((8, 4), dict(scaling="ntk_parts", factor=2.0))])
def test_rotary_tables_refusals(args, kw):
    from shadow_infer_b200.shadowkv import rotary_tables
    with pytest.raises(ValueError):
        rotary_tables(*args, device="cpu", **kw)


def test_argument_structs_match_the_header():
    """The sizes that the C compiler gives the argument structs (their fields are naturally aligned)."""
    import ctypes

    from shadow_infer_b200.shadowkv import paged_pool, rotary
    P, I, L = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64

    def struct_of(*fields):
        return type("S", (ctypes.Structure,), {"_fields_": [(str(i), f) for i, f in enumerate(fields)]})

    pool = struct_of(P, P, P, P, P, L, *[I] * 8)
    rows = struct_of(P, L, L, L, I, I)
    rope = struct_of(P, P, P, L, L, *[I] * 6)
    assert ctypes.sizeof(struct_of(*[rows] * 4, rope, I, I, I, I)) == rotary._ARGS.size
    assert ctypes.sizeof(struct_of(pool, *[rows] * 4, rope, P, P, P, I, I)) == paged_pool._APPEND.size
    assert ctypes.sizeof(struct_of(pool, rows, rows, P, P, P, I, I)) == paged_pool._READ.size
    assert ctypes.sizeof(struct_of(pool, rows, rows, P, P, P, L, P, I, I, ctypes.c_float, I)) == paged_pool._ATTENTION.size


def test_entry_points_refuse_before_a_launch():
    from shadow_infer_b200 import _lib
    from shadow_infer_b200.shadowkv import paged_pool, rotary
    lib = _lib.load()
    for f in (lib.skv_rotary, lib.skv_pool_append, lib.skv_pool_read, lib.skv_pool_attention):
        assert f(None, None) == _lib.SKV_ERR_INVALID_ARGUMENT
    none = (0,) * 6

    def rot(q, k=none, rope=(1, 1, 0, 0, 0, 0, 8, 4, 0, 0, 0), sizes=(1, 1, 8)):
        return lib.skv_rotary(rotary._ARGS.pack(*q, *k, *q, *k, *rope, *sizes, 0), None)

    assert rot((0, 8, 8, 8, 0, 1)) == _lib.SKV_ERR_INVALID_ARGUMENT                       # null rows
    assert rot((16, 8, 8, 8, 5, 1)) == _lib.SKV_ERR_INVALID_ARGUMENT                      # dtype
    assert rot((16, 8, 8, 8, 0, 1), rope=(1, 1, 0, 0, 0, 0, 7, 4, 0, 0, 0)) == _lib.SKV_ERR_SHAPE
    assert rot((16, 8, 8, 8, 0, 1), rope=(1, 1, 0, 0, 0, 0, 10, 4, 0, 0, 0)) == _lib.SKV_ERR_SHAPE
    assert rot((16, 8, 8, 8, 0, 1), rope=(0, 1, 0, 0, 0, 0, 8, 4, 0, 0, 0)) == _lib.SKV_ERR_INVALID_ARGUMENT
    assert rot((16, 8, 8, 8, 0, 1), rope=(1, 1, 1, 0, 0, 2, 8, 4, 0, 0, 0)) == _lib.SKV_ERR_INVALID_ARGUMENT
    assert rot((16, 8, 8, 8, 0, 1), (16, 8, 8, 8, 1, 1)) == _lib.SKV_ERR_SHAPE            # q and k of two types
    assert rot((16, 8, 8, 8, 0, 1), sizes=(1, 1, 0)) == _lib.SKV_ERR_INVALID_ARGUMENT
    assert rot((16, 8, 8, 8, 0, 1), sizes=(0, 1, 8)) == _lib.SKV_OK                       # nothing to do

    def attend(pool, q=(16, 8, 8, 8, 0, 2), out=(16, 8, 8, 8, 0, 2), lengths=1, scratch=16, need=1 << 30, S_q=1):
        return lib.skv_pool_attention(paged_pool._ATTENTION.pack(*pool, *q, *out, lengths, 0, scratch, need, 0, S_q, 0,
                                                                 1.0, 0), None)

    def pool(k=16, scale=0, table=16, N=4, P=8, H=2, D=8, G=0, precision=0, B=1):
        return (k, k, scale, scale, table, 4, 4, N, P, H, D, G, precision, B)

    bad = _lib.SKV_ERR_INVALID_ARGUMENT
    assert attend(pool(k=0)) == bad and attend(pool(table=0)) == bad and attend(pool(P=0)) == bad
    assert attend(pool(precision=4)) == bad and attend(pool(precision=2)) == bad and attend(pool(), lengths=0) == bad
    assert attend(pool(), scratch=0) == bad and attend(pool(), S_q=-1) == bad
    assert attend(pool(precision=3, scale=16, G=3)) == _lib.SKV_ERR_GROUP_SIZE
    assert attend(pool(H=3)) == _lib.SKV_ERR_SHAPE                                         # 2 query heads, 3 key heads
    assert attend(pool(), out=(16, 8, 8, 8, 1, 2)) == _lib.SKV_ERR_SHAPE
    assert attend(pool(), need=100) == _lib.SKV_ERR_SCRATCH
    assert attend(pool(D=4000)) == _lib.SKV_ERR_UNSUPPORTED
    assert attend(pool(B=0)) == _lib.SKV_OK and attend(pool(), S_q=0) == _lib.SKV_OK
    assert lib.skv_pool_attention_scratch_bytes(0) == 0 < lib.skv_pool_attention_scratch_bytes(128)


def test_no_cpu_fallback():
    if torch.cuda.is_available():
        pytest.skip("a CUDA device is present")
    from shadow_infer_b200.shadowkv import PagedKVPool, apply_rotary, paged_attention
    x = torch.zeros(1, 1, 1, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        apply_rotary(x, x[0, 0], x[0, 0])
    with pytest.raises(RuntimeError, match="CUDA"):
        paged_attention(x, x, x, torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="CUDA"):
        PagedKVPool(1, 1, 1, 8, 8)
    with pytest.raises(ValueError, match="precision"):
        PagedKVPool(1, 1, 1, 8, 8, precision="int3")
    with pytest.raises(ValueError, match=">= 1"):
        PagedKVPool(0, 1, 1, 8, 8)


def test_attention_refuses_only_what_tile_numbers_cannot_count():
    """One sequence whose table could hold more tiles than a launch counts is refused before any launch."""
    from shadow_infer_b200 import _lib
    from shadow_infer_b200.shadowkv import paged_pool
    lib = _lib.load()

    def attend(width, page, heads, S_q, D=128, dtype=0):
        pool = (16, 16, 0, 0, 16, width, width, 4, page, 1, D, 0, 0, 1)
        rows = (16, 0, 0, 0, dtype, heads)
        return lib.skv_pool_attention(paged_pool._ATTENTION.pack(*pool, *rows, *rows, 16, 0, 16, 1 << 40, 0, S_q, 0, 1.0, 0), None)

    assert attend(2 ** 26, 32, 1 << 14, 1 << 10) == _lib.SKV_ERR_TOO_LARGE
    assert "units" in _lib.last_error()


def test_attention_scratch_is_sized_by_device(monkeypatch):
    """The scratch a device needs depends on its SMs: what one device needed is not taken for another's."""
    from types import SimpleNamespace

    from shadow_infer_b200.shadowkv import paged_pool
    sms = iter((100, 160))
    fake = SimpleNamespace(skv_pool_attention_scratch_bytes=lambda D: next(sms) * D, skv_pool_attention_scratch_zeros=lambda: 16)
    monkeypatch.setattr(paged_pool._lib, "load", lambda: fake)
    monkeypatch.setattr(paged_pool, "_capturing", lambda: False)
    monkeypatch.setattr(paged_pool, "_SCRATCH", {})
    monkeypatch.setattr(paged_pool, "_SCRATCH_BYTES", {})
    got = [paged_pool._scratch(torch.device("meta", i), 7, 128).numel() for i in (0, 1, 0, 1)]
    assert got == [12800, 20480, 12800, 20480]


def test_rows_that_31_bits_do_not_number_are_refused():
    from shadow_infer_b200 import _lib
    from shadow_infer_b200.shadowkv import paged_pool, rotary
    lib = _lib.load()
    rows, none = (16, 0, 0, 0, 0, 1), (0,) * 6
    for S in (2 ** 31 - 1, 2 ** 31 - 10):
        assert lib.skv_rotary(rotary._ARGS.pack(*rows, *none, *rows, *none, 16, 16, 0, 0, 0, 0, 8, 4, 0, 0, 0, 1, S, 8, 0),
                              None) == _lib.SKV_ERR_TOO_LARGE
        pool = (16, 16, 0, 0, 16, 4, 4, 4, 8, 1, 8, 0, 0, 1)
        assert lib.skv_pool_read(paged_pool._READ.pack(*pool, *rows, *rows, 0, 16, 0, S, 0), None) == _lib.SKV_ERR_TOO_LARGE


def test_attention_refuses_scratch_between_16_byte_boundaries():
    """Parts go to the scratch 16 bytes at a time."""
    from shadow_infer_b200 import _lib
    from shadow_infer_b200.shadowkv import paged_pool
    lib = _lib.load()
    pool, rows = (16, 16, 0, 0, 16, 4, 4, 4, 8, 2, 8, 0, 0, 1), (16, 8, 8, 8, 0, 2)
    for scratch in (4, 24, 40):   # (with too few bytes too: nothing is launched either way)
        args = paged_pool._ATTENTION.pack(*pool, *rows, *rows, 16, 0, scratch, 100, 0, 1, 0, 1.0, 0)
        assert lib.skv_pool_attention(args, None) == _lib.SKV_ERR_INVALID_ARGUMENT
        assert "boundary" in _lib.last_error()
