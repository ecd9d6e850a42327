"""Refusals of the serving-step operators (chunk attention, rotary positions, page upkeep): every
case is rejected, or found empty, on the host before anything is launched, so no GPU is needed."""
import ctypes as C

import pytest

from kvx_b200 import abi

OK, INVALID, UNSUPPORTED = abi.STATUS_OK, abi.STATUS_INVALID_ARGUMENT, abi.STATUS_UNSUPPORTED
FAKE = 0x10000  # a non-NULL "device" address that is never dereferenced on these paths
OUT = 0x20000   # another one


def cache(dtype=abi.DTYPE_BF16, layout=abi.LAYOUT_NHD, pack=1, dim=64):
    return abi.cache_desc(abi.CacheGeometry(8, 16, 2, dim, layout, pack), dtype, FAKE, FAKE)


def mutated(desc, **kw):
    for path, value in kw.items():
        at = desc
        *way, last = path.split("__")
        for name in way:
            at = at[int(name)] if name.isdigit() else getattr(at, name)
        if last.isdigit():
            at[int(last)] = value
        else:
            setattr(at, last, value)
    return desc


# ---------------------------------------------------------------- chunk attention

def chunk(**kw):
    return mutated(abi.chunk_attention_desc(3, 10, 8, 64, abi.DTYPE_BF16, FAKE, OUT, 0.1, True, 64, abi.DTYPE_S32, FAKE, 4, FAKE,
                                            abi.DTYPE_S32, FAKE), **kw)


def attend(L, c, a, ws=FAKE, nbytes=1 << 30, scales=True):
    s = abi.scale_desc(FAKE if scales else None, abi.SCALE_PER_TENSOR, 2)
    return L.kvx_launch_paged_attention_chunk(C.byref(c) if c is not None else None, C.byref(a) if a is not None else None, C.byref(s),
                                              C.byref(s), ws, nbytes, None)


def test_chunk_attention_refusals(built_lib):
    L = built_lib
    assert attend(L, None, chunk()) == INVALID and attend(L, cache(), None) == INVALID
    need = L.kvx_paged_attention_chunk_workspace_bytes(3, 10, 8, 2, 64, 64)
    assert need > 0
    assert attend(L, cache(), chunk(), None, need) == INVALID
    assert attend(L, cache(), chunk(), FAKE, need - 1) == INVALID
    assert attend(L, cache(), chunk(), FAKE + 8, need) == INVALID
    for kw in (dict(size=8), dict(num_q_heads=7), dict(num_q_heads=0), dict(max_seq_len=0), dict(causal=2), dict(block_table__size=4),
               dict(seq_lens__size=4), dict(seq_lens__seq_count=2), dict(seq_lens__dtype=abi.DTYPE_S64), dict(query__shape__1=6),
               dict(query__shape__2=32), dict(out__shape__0=9), dict(query__ndim=2), dict(query__size=8),
               dict(query_indptr_dtype=abi.DTYPE_U32), dict(query_indptr=None), dict(query__data=None), dict(out__data=None), dict(out__data=FAKE),
               dict(block_table__indices=None), dict(seq_lens__lengths=None), dict(block_table__max_blocks_per_seq=0),
               dict(max_seq_len=2 ** 31)):
        assert attend(L, cache(), chunk(**kw)) == INVALID, kw
    for kw in (dict(block_table__format=abi.TABLE_RAGGED), dict(out__dtype=abi.DTYPE_F16), dict(query__dtype=abi.DTYPE_F16),
               dict(query__dtype=abi.DTYPE_S32, out__dtype=abi.DTYPE_S32), dict(query__stride__0=100), dict(query__stride__1=65),
               dict(out__stride__2=2)):
        assert attend(L, cache(), chunk(**kw)) == UNSUPPORTED, kw
    c = cache()
    c.v.dtype = abi.DTYPE_F16
    assert attend(L, c, chunk()) == INVALID
    assert attend(L, cache(abi.DTYPE_F8_E4M3), chunk(), scales=False) == UNSUPPORTED
    assert attend(L, mutated(cache(), k__layout=abi.LAYOUT_CUSTOM, v__layout=abi.LAYOUT_CUSTOM), chunk()) == UNSUPPORTED
    wide = abi.chunk_attention_desc(3, 10, 8, 1100, abi.DTYPE_BF16, FAKE, OUT, 0.1, True, 64, abi.DTYPE_S32, FAKE, 4, FAKE, abi.DTYPE_S32, FAKE)
    assert attend(L, cache(dim=1100), wide) == UNSUPPORTED
    many = abi.chunk_attention_desc(3, 2 ** 30, 8, 64, abi.DTYPE_BF16, FAKE, OUT, 0.1, True, 64, abi.DTYPE_S32, FAKE, 4, FAKE, abi.DTYPE_S32, FAKE)
    assert attend(L, cache(), many) == UNSUPPORTED  # 2^30 rows x 4 heads
    # nothing to do
    none = abi.chunk_attention_desc(3, 0, 8, 64, abi.DTYPE_BF16, 0, 0, 0.1, True, 64, abi.DTYPE_S32, FAKE, 4, FAKE, abi.DTYPE_S32, FAKE)
    assert attend(L, cache(), none, None, 0) == OK
    none = abi.chunk_attention_desc(0, 5, 8, 64, abi.DTYPE_BF16, FAKE, OUT, 0.1, True, 64, abi.DTYPE_S32, 0, 4, 0, abi.DTYPE_S32, FAKE)
    assert attend(L, cache(), none, None, 0) == OK


def test_chunk_workspace_is_bounded(built_lib):
    """Scratch does not grow with the context, and little with the batch."""
    f = built_lib.kvx_paged_attention_chunk_workspace_bytes
    assert f(0, 5, 8, 2, 64, 64) == 0 and f(1, 0, 8, 2, 64, 64) == 0
    assert f(1, 4, 32, 8, 128, 1 << 20) == f(1, 4, 32, 8, 128, 1 << 30)
    assert f(512, 1 << 20, 32, 8, 128, 1 << 20) < 50 << 20
    assert f(1, 17, 32, 4, 64, 64) < 4096  # too short to be cut


# ---------------------------------------------------------------- rotary positions

def rotary(with_key=True, tokens=4, **kw):
    r = abi.RotaryDesc()
    r.size = C.sizeof(abi.RotaryDesc)
    r.rotary_dim, r.position_dtype, r.positions, r.inv_freq, r.factor = 64, abi.DTYPE_S64, FAKE, FAKE, 1.0
    for name, heads in (("query", 8), ("query_out", 8)) + ((("key", 2), ("key_out", 2)) if with_key else ()):
        setattr(r, name, abi.tensor_desc(FAKE, abi.DTYPE_BF16, (tokens, heads, 64), layout=abi.LAYOUT_INVALID))
    return mutated(r, **kw)


def test_rotary_refusals(built_lib):
    turn = lambda r: built_lib.kvx_launch_rotary(C.byref(r) if r is not None else None, None)
    assert turn(None) == INVALID
    for kw in (dict(size=8), dict(rotary_dim=3), dict(rotary_dim=66), dict(flags=4), dict(position_dtype=abi.DTYPE_U32),
               dict(positions=None), dict(inv_freq=None), dict(query_out__data=None), dict(key_out__data=None), dict(query__ndim=4),
               dict(query_out__shape__1=7), dict(key__shape__0=5), dict(key__shape__2=32), dict(query__size=8)):
        assert turn(rotary(**kw)) == INVALID, kw
    for kw in (dict(query__dtype=abi.DTYPE_F8_E4M3), dict(query_out__dtype=abi.DTYPE_F16), dict(key__dtype=abi.DTYPE_F16),
               dict(query__stride__1=65), dict(query__stride__2=2), dict(key_out__stride__0=64)):
        assert turn(rotary(**kw)) == UNSUPPORTED, kw
    assert turn(rotary(tokens=0)) == OK
    empty = rotary(with_key=False, tokens=0, query__data=None, query_out__data=None)
    assert turn(empty) == OK
    assert turn(rotary(with_key=False, query__data=None)) == INVALID


def test_rotary_write_refusals(built_lib):
    def write(**kw):
        w = abi.write_desc(4, 2, 64, abi.DTYPE_BF16, FAKE, FAKE, abi.DTYPE_S64, FAKE)
        return mutated(w, **kw)

    def go(c=None, w=None, r=None):
        c, w, r = c or cache(), w or write(), r or rotary(with_key=False)
        return built_lib.kvx_launch_rotary_write_kv(C.byref(c), C.byref(w), C.byref(r), None)

    assert built_lib.kvx_launch_rotary_write_kv(None, None, None, None) == INVALID
    assert go(r=rotary(with_key=True)) == INVALID  # the keys come from the write descriptor
    for kw in (dict(size=8), dict(io__size=8), dict(slots__size=4), dict(io__head_dim=32), dict(io__num_kv_heads=3), dict(slots__token_count=3),
               dict(io__key__shape__0=5), dict(slots__dtype=abi.DTYPE_U32), dict(slots__slots=None), dict(io__key__data=None),
               dict(io__value__data=None)):
        assert go(w=write(**kw)) == INVALID, kw
    for kw in (dict(io__value__dtype=abi.DTYPE_F16), dict(io__key__stride__0=64), dict(io__value__stride__1=65)):
        assert go(w=write(**kw)) == UNSUPPORTED, kw
    assert go(c=cache(abi.DTYPE_F16)) == UNSUPPORTED
    assert go(c=cache(abi.DTYPE_F8_E4M3)) == UNSUPPORTED  # no scales
    assert go(c=mutated(cache(), k__layout=abi.LAYOUT_CUSTOM, v__layout=abi.LAYOUT_CUSTOM)) == UNSUPPORTED
    assert go(r=rotary(with_key=False, tokens=5)) == INVALID
    assert go(r=rotary(with_key=False, rotary_dim=128)) == INVALID
    w = abi.write_desc(0, 2, 64, abi.DTYPE_BF16, 0, 0, abi.DTYPE_S64, 0)
    assert go(w=w, r=rotary(with_key=False, tokens=0)) == OK


# ---------------------------------------------------------------- page upkeep

def test_copy_pages_refusals(built_lib):
    def go(caches, n=4, code=abi.DTYPE_S32, src=FAKE, dst=FAKE, ws=None, nbytes=0):
        arr = (abi.CacheDesc * max(1, len(caches)))(*caches)
        return built_lib.kvx_launch_copy_pages(arr, len(caches), src, dst, code, n, ws, nbytes, None)

    assert go([cache()], code=abi.DTYPE_U32) == INVALID
    assert go([cache()], src=None) == INVALID and go([cache()], dst=None) == INVALID
    assert go([mutated(cache(), size=8)]) == INVALID
    assert go([mutated(cache(), block_size=0)]) == INVALID
    assert go([cache(), mutated(cache(), num_blocks=7)]) == INVALID
    assert go([mutated(cache(), v__dtype=abi.DTYPE_F16)]) == INVALID
    assert go([mutated(cache(), k__data=None)]) == INVALID
    assert go([mutated(cache(), k__dtype=abi.DTYPE_INVALID, v__dtype=abi.DTYPE_INVALID)]) == UNSUPPORTED
    assert go([mutated(cache(), v__layout=abi.LAYOUT_CUSTOM)]) == UNSUPPORTED
    need = built_lib.kvx_copy_pages_workspace_bytes(1000)
    assert need >= 1000 and built_lib.kvx_copy_pages_workspace_bytes(100) == 0
    assert go([cache()], n=1000) == INVALID
    assert go([cache()], n=1000, ws=FAKE, nbytes=need - 1) == INVALID
    assert go([cache()], n=0, src=None, dst=None) == OK
    assert go([], n=4) == OK


def test_table_plans_refuse(built_lib):
    L = built_lib
    table = lambda **kw: mutated(abi.block_table_desc(4, 8, abi.DTYPE_S32, FAKE), **kw)
    lens = lambda **kw: mutated(abi.seq_lens_desc(4, abi.DTYPE_S32, FAKE), **kw)

    def free(t=None, s=None, refs=FAKE, rows=FAKE, n=2):
        return L.kvx_launch_free_sequences(C.byref(t or table()), C.byref(s or lens()), refs, 16, rows, n, None)

    def fork(t=None, s=None, refs=FAKE, bs=16, a=FAKE, b=FAKE, n=2, src=FAKE, dst=FAKE, ws=FAKE, nbytes=1 << 20):
        return L.kvx_launch_fork_sequences(C.byref(t or table()), C.byref(s or lens()), refs, 16, bs, a, b, n, src, dst, ws, nbytes, None)

    def compact(t=None, refs=FAKE, src=FAKE, dst=FAKE):
        return L.kvx_launch_compact_pages(C.byref(t or table()), refs, 16, src, dst, None)

    for f in (free, fork, compact):
        assert f(t=table(size=4)) == INVALID
        assert f(t=table(format=abi.TABLE_RAGGED)) == UNSUPPORTED
        assert f(t=table(index_dtype=abi.DTYPE_U32)) == INVALID
        assert f(t=table(indices=None)) == INVALID
        assert f(refs=None) == INVALID
    for f in (free, fork):
        assert f(s=lens(size=4)) == INVALID
        assert f(s=lens(dtype=abi.DTYPE_S64)) == INVALID
        assert f(s=lens(seq_count=3)) == INVALID
        assert f(s=lens(lengths=None)) == INVALID
    assert L.kvx_launch_free_sequences(C.byref(table()), None, FAKE, 16, FAKE, 2, None) == INVALID
    assert free(rows=None) == INVALID and free(rows=None, n=0) == OK
    assert fork(bs=0) == INVALID and fork(a=None) == INVALID and fork(b=None) == INVALID
    assert fork(src=None) == INVALID and fork(dst=None) == INVALID and fork(ws=None) == INVALID
    assert fork(nbytes=L.kvx_fork_workspace_bytes(2) - 1) == INVALID
    assert fork(n=0, a=None, b=None) == OK
    assert compact(src=None) == INVALID and compact(dst=None) == INVALID


def test_python_front_end_refuses(built_lib):
    """Wrong shapes, types and devices raise before the library is called."""
    import torch
    from kvx_b200 import ops
    q = torch.zeros((4, 8, 64))
    for call in (lambda: ops.rotary_embedding(q, None, torch.zeros(4, dtype=torch.int64), torch.ones(32, dtype=torch.float64)),
                 lambda: ops.rotary_embedding(q[0], None, torch.zeros(4, dtype=torch.int64), torch.ones(32, dtype=torch.float64)),
                 lambda: ops.rotary_and_cache(q, q, q, torch.zeros(4, dtype=torch.int64), torch.ones(32, dtype=torch.float64), q, q,
                                              torch.zeros(4, dtype=torch.int64)),
                 lambda: ops.copy_pages([], [], torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)),
                 lambda: ops.copy_pages([q], [q], torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)),
                 lambda: ops.compact_pages(torch.zeros((2, 2), dtype=torch.int32), torch.zeros(4, dtype=torch.int32)),
                 lambda: ops.free_sequences(torch.zeros((2, 2), dtype=torch.int32), torch.zeros(2, dtype=torch.int32),
                                            torch.zeros(4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)),
                 lambda: ops.paged_attention_chunk(q, q, q, torch.zeros((1, 1), dtype=torch.int32), torch.zeros(1, dtype=torch.int32),
                                                   torch.zeros(2, dtype=torch.int32), 0.1),
                 lambda: ops.paged_attention_chunk(q, q, q, torch.zeros((1, 1), dtype=torch.int32), torch.zeros(1, dtype=torch.int32),
                                                   torch.zeros(3, dtype=torch.int32), 0.1)):
        with pytest.raises((ValueError, TypeError)):
            call()
    for bad in (dict(rotary_dim=3), dict(rotary_dim=0), dict(rotary_dim=64, scaling="other"), dict(rotary_dim=64, scale=0.0),
                dict(rotary_dim=64, base=1.0), dict(rotary_dim=2, scaling="ntk"), dict(rotary_dim=64, scaling="bands", low=4.0, high=1.0)):
        with pytest.raises(ValueError):
            ops.rotary_inv_freq(**bad)
