"""CPU-only checks of page bounds, page selection, beam selection and reordering: argument structs, and the refusals made before any
launch."""

import ctypes

import pytest
import torch


def test_argument_structs_match_the_header():
    """The sizes that the C compiler gives the argument structs (their fields are naturally aligned)."""
    from shadow_infer_b200.shadowkv import beam, page_selection, paged_pool
    P, I, L, F = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float

    def struct_of(*fields):
        return type("S", (ctypes.Structure,), {"_fields_": [(str(i), f) for i, f in enumerate(fields)]})

    pool = struct_of(P, P, P, P, P, L, *[I] * 8)
    rows = struct_of(P, L, L, L, I, I)
    attention = struct_of(pool, rows, rows, P, P, P, L, P, I, I, F, I)
    assert ctypes.sizeof(struct_of(pool, *[P] * 5)) == page_selection._BOUNDS.size
    assert ctypes.sizeof(struct_of(rows, *[P] * 8, L, L, *[I] * 12)) == page_selection._SELECT.size
    assert ctypes.sizeof(struct_of(attention, P, L, L, L, P, L, I, I)) == paged_pool._SPARSE.size
    assert ctypes.sizeof(struct_of(P, L, L, *[P] * 6, L, *[I] * 6)) == beam._BEAM.size
    assert ctypes.sizeof(struct_of(pool, *[P] * 7, I, I)) == beam._REORDER.size


def _pool(k=16, scale=0, table=16, N=4, P=8, H=2, D=8, G=0, precision=0, B=1, width=4):
    return (k, k, scale, scale, table, width, width, N, P, H, D, G, precision, B)


def test_bounds_refuse_before_a_launch():
    from shadow_infer_b200 import _lib
    from shadow_infer_b200.shadowkv import page_selection
    lib = _lib.load()
    bad = _lib.SKV_ERR_INVALID_ARGUMENT

    def bounds(pool, lengths=16, out=16, steps=16):
        return lib.skv_pool_bounds(page_selection._BOUNDS.pack(*pool, 0, lengths, out, steps, 0), None)

    assert lib.skv_pool_bounds(None, None) == bad
    assert bounds(_pool(k=0)) == bad and bounds(_pool(table=0)) == bad and bounds(_pool(P=0)) == bad and bounds(_pool(D=0)) == bad
    assert bounds(_pool(), lengths=0) == bad and bounds(_pool(), out=0) == bad and bounds(_pool(), steps=0) == bad
    assert bounds(_pool(precision=2)) == bad                                              # no scales
    assert bounds(_pool(precision=3, scale=16, G=3)) == _lib.SKV_ERR_GROUP_SIZE
    assert bounds(_pool(B=0), lengths=0) == _lib.SKV_OK and bounds(_pool(N=0, k=0)) == _lib.SKV_OK


def test_select_refuses_before_a_launch():
    from shadow_infer_b200 import _lib
    from shadow_infer_b200.shadowkv import page_selection
    lib = _lib.load()
    bad, large = _lib.SKV_ERR_INVALID_ARGUMENT, _lib.SKV_ERR_TOO_LARGE

    def select(q=(16, 8, 8, 8, 0, 2), ptrs=(16, 16, 16, 16, 0, 16, 16, 0), room=1 << 40, width=4, N=4, P=8, H=2, D=8, B=1, S=1,
               keep=3, first=1, recent=1):
        return lib.skv_pool_select(page_selection._SELECT.pack(*q, *ptrs, width, room, width, N, P, H, D, B, S, keep, first, recent, 0, 0),
                                   None)

    assert lib.skv_pool_select(None, None) == bad
    assert select(keep=0) == bad and select(recent=0) == bad and select(first=-1) == bad and select(first=2, recent=2) == bad
    assert select(first=2 ** 31 - 1, recent=1) == bad
    assert select(P=0) == bad and select(H=0) == bad and select(D=0) == bad and select(S=-1) == bad and select(B=-1) == bad
    for i in (0, 1, 2, 3, 5, 6):
        assert select(ptrs=tuple(0 if j == i else p for j, p in enumerate((16, 16, 16, 16, 0, 16, 16, 0)))) == bad
    assert select(q=(0, 8, 8, 8, 0, 2)) == bad and select(q=(16, 8, 8, 8, 7, 2)) == bad
    assert select(q=(16, 8, 8, 8, 0, 3)) == _lib.SKV_ERR_SHAPE
    assert select(D=1032) == _lib.SKV_ERR_UNSUPPORTED
    assert select(B=1 << 20) == large and select(S=1 << 30) == large and select(H=1 << 17, q=(16, 8, 8, 8, 0, 1 << 17)) == large
    assert select(width=(1 << 30) + 1) == large
    assert select(room=15) == _lib.SKV_ERR_SCRATCH
    assert select(B=0) == _lib.SKV_OK and select(S=0) == _lib.SKV_OK
    assert lib.skv_pool_select_scratch_bytes(3, 2, 5, 7) >= 3 * 2 * 5 * 7 * 4 and lib.skv_pool_select_scratch_bytes(-1, 2, 5, 7) == 0


def test_sparse_attention_refuses_before_a_launch():
    from shadow_infer_b200 import _lib
    from shadow_infer_b200.shadowkv import paged_pool
    lib = _lib.load()
    bad = _lib.SKV_ERR_INVALID_ARGUMENT

    def attend(pool=None, q=(16, 16, 8, 16, 0, 2), out=(16, 16, 8, 16, 0, 2), lengths=16, S=1, pages=16, tables=128, room=1 << 20, keep=4):
        return lib.skv_pool_sparse_attention(
            paged_pool._SPARSE.pack(*(pool or _pool()), *q, *out, lengths, 0, 16, 1 << 40, 0, S, 0, 1.0, 0, pages, 8, 4, 8, tables, room,
                                    keep, 0), None)

    assert lib.skv_pool_sparse_attention(None, None) == bad
    assert attend(pages=0) == bad and attend(tables=0) == bad and attend(tables=192) == bad and attend(keep=0) == bad and attend(lengths=0) == bad
    assert attend(q=(0, 16, 8, 16, 0, 2)) == bad and attend(_pool(P=0)) == bad
    assert attend(room=4) == _lib.SKV_ERR_SCRATCH
    assert attend(_pool(N=1 << 30, H=4), q=(16, 32, 8, 32, 0, 4), out=(16, 32, 8, 32, 0, 4)) == _lib.SKV_ERR_TOO_LARGE
    assert attend(_pool(B=1 << 23, H=4), q=(16, 32, 8, 32, 0, 4), out=(16, 32, 8, 32, 0, 4)) == _lib.SKV_ERR_TOO_LARGE
    # two new tokens whose heads are not between them
    assert attend(S=2, q=(16, 32, 16, 8, 0, 2), out=(16, 32, 16, 8, 0, 2)) == _lib.SKV_ERR_UNSUPPORTED
    assert attend(S=2, q=(16, 32, 8, 16, 0, 2), out=(16, 32, 16, 8, 0, 2)) == _lib.SKV_ERR_UNSUPPORTED
    assert attend(_pool(B=0)) == _lib.SKV_OK and attend(S=0) == _lib.SKV_OK


def test_beam_refuses_before_a_launch():
    from shadow_infer_b200 import _lib
    from shadow_infer_b200.shadowkv import beam
    lib = _lib.load()
    bad, large = _lib.SKV_ERR_INVALID_ARGUMENT, _lib.SKV_ERR_TOO_LARGE

    def select(logits=16, scores=16, finished=0, outs=(16, 16, 16), scratch=16, room=0, dtype=0, B=1, beams=4, V=100, keep=4, pad=0):
        return lib.skv_beam_select(beam._BEAM.pack(logits, 400, 100, scores, finished, *outs, scratch, room, dtype, B, beams, V, keep, pad),
                                   None)

    assert lib.skv_beam_select(None, None) == bad
    assert select() == _lib.SKV_ERR_SCRATCH                                               # all else is right
    for wrong in (dict(logits=0), dict(scores=0), dict(outs=(0, 16, 16)), dict(outs=(16, 0, 16)), dict(outs=(16, 16, 0)), dict(scratch=0),
                  dict(scratch=8), dict(logits=18), dict(B=-1), dict(beams=0), dict(V=0), dict(keep=0), dict(dtype=3),
                  dict(finished=16, pad=100), dict(finished=16, pad=-1)):
        assert select(**wrong) == bad, wrong
    assert select(logits=17, dtype=1) == bad and select(logits=18, dtype=1) == _lib.SKV_ERR_SCRATCH
    assert select(keep=401) == _lib.SKV_ERR_SHAPE
    assert select(keep=129) == large and select(beams=4097) == large and select(V=2 ** 31 - 1, beams=1) == large
    assert select(B=0) == _lib.SKV_OK
    assert lib.skv_beam_scratch_bytes(0, 4, 100, 4) == 0 == lib.skv_beam_scratch_bytes(1, 5000, 100, 4)


def test_reorder_refuses_before_a_launch():
    from shadow_infer_b200 import _lib
    from shadow_infer_b200.shadowkv import beam
    lib = _lib.load()
    bad = _lib.SKV_ERR_INVALID_ARGUMENT

    def reorder(pool, lengths=16, parents=16, table=16, new=16, bounds=0, steps=0, size=8, beams=2):
        return lib.skv_pool_reorder(beam._REORDER.pack(*pool, lengths, parents, table, new, bounds, steps, 0, size, beams), None)

    assert lib.skv_pool_reorder(None, None) == bad
    good = _pool(B=4)
    assert reorder(_pool(B=4, k=0)) == bad and reorder(good, lengths=0) == bad and reorder(good, parents=0) == bad
    assert reorder(good, table=0) == bad and reorder(good, new=0) == bad and reorder(good, bounds=16) == bad and reorder(good, steps=16) == bad
    assert reorder(good, size=2) == bad
    assert reorder(good, beams=0) == _lib.SKV_ERR_SHAPE and reorder(good, beams=3) == _lib.SKV_ERR_SHAPE
    assert reorder(_pool(B=2048), beams=2048) == _lib.SKV_ERR_TOO_LARGE and reorder(_pool(B=4, H=40000)) == _lib.SKV_ERR_TOO_LARGE
    assert reorder(_pool(B=0), lengths=0) == _lib.SKV_OK


def test_python_refusals_before_any_device():
    from shadow_infer_b200.shadowkv import beam_select, paged_reorder
    x = torch.zeros(2, 3, 5)
    for args, kw in (((x[0], x[0]), {}), ((x, torch.zeros(2, 2)), {}), ((x, torch.zeros(2, 3), 0), {}), ((x, torch.zeros(2, 3), 16), {}),
                     ((torch.zeros(1, 1, 500), torch.zeros(1, 1), 129), {}), ((x[:, :0], torch.zeros(2, 0)), {}),
                     ((x, torch.zeros(2, 3)), dict(finished=torch.zeros(2, 2, dtype=torch.bool))),
                     ((x, torch.zeros(2, 3)), dict(finished=torch.zeros(2, 3))),
                     ((x, torch.zeros(2, 3)), dict(finished=torch.zeros(2, 3, dtype=torch.bool), pad_token=5))):
        with pytest.raises(ValueError):
            beam_select(*args, **kw)
    with pytest.raises(ValueError, match="parents"):
        paged_reorder(x, x, x, x, torch.zeros(3))
    with pytest.raises(ValueError, match="int32 or int64"):
        paged_reorder(x, x, x, x, torch.zeros(3, 2))


def test_no_cpu_fallback():
    if torch.cuda.is_available():
        pytest.skip("a CUDA device is present")
    from shadow_infer_b200.shadowkv import beam_select, page_bounds, page_select, paged_reorder
    x, table, lens = torch.zeros(1, 1, 1, 8), torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        page_bounds(x, table, lens)
    with pytest.raises(RuntimeError, match="CUDA"):
        page_select(x, torch.zeros(1, 1, 2, 8, dtype=torch.int8), torch.ones(1, 1), table, lens, 1, 2)
    with pytest.raises(RuntimeError, match="CUDA"):
        beam_select(x[0], torch.zeros(1, 1))
    with pytest.raises(RuntimeError, match="CUDA"):
        paged_reorder(x, x, table, lens, torch.zeros(1, 1, dtype=torch.int64))
