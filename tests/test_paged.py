"""The paged kernels' checks on the host: what each binding of page_plan, rope_pages, attention_pages and
logits_pick must hold, and the params they refuse, before any device is touched."""

import numpy as np
import pytest

SPARE = 0xFFFFFFFF


def plan(pkg, **kw):
    return pkg.TgParams(**{**dict(seqs=5, rows=40, stride=6, n=20, capacity=32, slots=64, first=100), **kw})


def heads(pkg, **kw):
    base = dict(dtype=pkg.BF16, heads=16, kv_heads=2, head_dim=64, rows=7, capacity=32, slots=64)
    return pkg.TgParams(**{**base, **kw})


def pick(pkg, **kw):
    return pkg.TgParams(**{**dict(dtype=pkg.F32, rows=3, n=1000, stride=1008, k=50, k1=4, m=2), **kw})


def test_page_plan_bindings(pkg):
    assert pkg.needs("page_plan", plan(pkg)) == [20, 20, 80, 120, 320, 160, 24, 20, 16]
    assert pkg.needs("page_plan", plan(pkg, n=0))[2] == 16


@pytest.mark.parametrize("kw", [dict(seqs=0), dict(seqs=16385), dict(rows=0), dict(stride=0), dict(capacity=0), dict(capacity=24),
                                dict(slots=0), dict(capacity=1 << 16, slots=1 << 16), dict(rows=1 << 31)])
def test_page_plan_refuses(pkg, kw):
    with pytest.raises(pkg.ShapeError):
        pkg.needs("page_plan", plan(pkg, **kw))


def test_rope_pages_bindings(pkg):
    p = heads(pkg, rope=1, k=32, n=500)
    cache = 64 * 2 * 32 * 64 * 2
    assert pkg.needs("rope_pages", p) == [56, 28, 7 * 20 * 64 * 4, 500 * 16 * 4, 500 * 16 * 4, 7 * 16 * 64 * 2, cache, cache]
    p.flags = 2
    assert pkg.needs("rope_pages", p)[2] == 7 * 20 * 64 * 2
    p = heads(pkg, rope=0, dtype=0)
    assert pkg.needs("rope_pages", p)[3:6] == [16, 16, 7 * 16 * 64 * 4]


@pytest.mark.parametrize("kw", [dict(k=0), dict(k=3), dict(k=66), dict(n=0), dict(rope=0), dict(flags=4), dict(heads=0), dict(kv_heads=0),
                                dict(heads=15), dict(heads=32), dict(head_dim=96), dict(rows=0), dict(dtype=2), dict(dtype=7),
                                dict(capacity=8), dict(slots=0)])
def test_rope_pages_refuses(pkg, kw):
    with pytest.raises(pkg.ShapeError):
        pkg.needs("rope_pages", heads(pkg, **{**dict(rope=1, k=32, n=500), **kw}))


def test_attention_pages_bindings(pkg):
    p = heads(pkg, first=100, seqs=5, stride=6)
    got, cache = pkg.needs("attention_pages", p), 64 * 2 * 32 * 64 * 2
    assert got[:6] + got[7:] == [7 * 16 * 64 * 2, cache, cache, 56, 120, 16, 7 * 16 * 64 * 2]
    assert got[6] == pkg.attention_pages_work(p) > 0
    p.first = 129
    assert pkg.needs("attention_pages", p)[5] == 20
    p.first = 0
    assert pkg.needs("attention_pages", p)[5] == 16
    # The work grows with the rows alone, not with what runs beside them.
    p.rows = 14
    p7 = heads(pkg, first=0, seqs=5, stride=6)
    fixed = 256  # its alignment
    assert pkg.attention_pages_work(p) - fixed == 2 * (pkg.attention_pages_work(p7) - fixed)


@pytest.mark.parametrize("kw", [dict(seqs=0), dict(stride=0), dict(rows=0), dict(rows=65536), dict(first=SPARE), dict(heads=18),
                                dict(head_dim=32), dict(dtype=2), dict(capacity=40), dict(slots=0), dict(heads=2048, kv_heads=512)])
def test_attention_pages_refuses(pkg, kw):
    with pytest.raises(pkg.ShapeError):
        pkg.needs("attention_pages", heads(pkg, **{**dict(first=100, seqs=5, stride=6), **kw}))


def test_logits_pick_bindings(pkg):
    assert pkg.needs("logits_pick", pick(pkg)) == [12096, 200, 72, 36, 16, 16, 2 * 32 * 4, 12096, 12]
    assert pkg.needs("logits_pick", pick(pkg, dtype=1, k=0, k1=0, m=0)) == [6048, 16, 72, 36, 16, 16, 16, 6048, 12]


@pytest.mark.parametrize("kw", [dict(n=0), dict(stride=999), dict(rows=0), dict(rows=65536), dict(dtype=2), dict(n=1 << 31, stride=1 << 31),
                                dict(k=1 << 30)])
def test_logits_pick_refuses(pkg, kw):
    with pytest.raises(pkg.ShapeError):
        pkg.needs("logits_pick", pick(pkg, **kw))


def test_unknown_kernels_and_null_handles(pkg):
    import ctypes

    with pytest.raises(pkg.InvalidError):
        pkg.needs("page_plans", plan(pkg))
    count = ctypes.c_size_t()
    for kernel in (13, 31, 1008):
        assert pkg.library().tg_dispatch_needs(kernel, ctypes.byref(plan(pkg)), None, 0, ctypes.byref(count)) == 1
    assert pkg.library().tg_dispatch_needs(27, None, None, 0, ctypes.byref(count)) == 1
    assert pkg.library().tg_call_enqueue(None, None) == 1
    assert pkg.library().tg_call_create(None, None, None) == 1
    assert pkg.library().tg_call_destroy(None) == 0
    out = ctypes.c_void_p()
    assert pkg.library().tg_mem_wrap(None, 16, 16, ctypes.byref(out)) == 1


def test_a_strided_tensor_is_not_wrapped(pkg):
    class Strided:
        nbytes = 64

        def is_contiguous(self):
            return False

    with pytest.raises(pkg.ShapeError):
        pkg.Memory.wrap(None, Strided())


def test_the_rest_of_the_table_tells_its_bindings_too(pkg, syn):
    shape = syn.shape_of(syn.S05B, capacity=64)
    p = pkg.params(shape, "bf16", rows=2, slots=2)
    assert pkg.needs("rmsnorm", p) == [2 * 1024 * 4, 1024 * 4, 2 * 1024 * 4]
    assert np.all(np.array(pkg.needs("rope_rows", p)) > 0)


@pytest.mark.parametrize("count", [1, 2, 3])
def test_arrays_of_few_entries_hold_those_alone(pkg, count):
    """16 bytes stand in for an array without entries; one to three entries are four bytes each."""
    assert pkg.needs("page_plan", plan(pkg, n=count))[2] == 4 * count
    assert pkg.needs("attention_pages", heads(pkg, first=32 * count, seqs=5, stride=6))[5] == 4 * count
    assert pkg.needs("rope_pages", heads(pkg, rope=1, k=2, n=count))[3:5] == [4 * count, 4 * count]
    assert pkg.needs("logits_pick", pick(pkg, k=count))[1] == 4 * count
    assert pkg.needs("logits_pick", pick(pkg, k1=count))[4:6] == [4 * count, 4 * count]
    assert pkg.needs("logits_pick", pick(pkg, n=32 * count, m=1))[6] == 4 * count
    assert pkg.needs("logits_pick", pick(pkg, n=30, m=count))[6] == 4 * count
