"""CPU: what the decode entry points refuse before they touch a device, through the C ABI."""
import ctypes

import pytest

import welvet.cuda_b200 as W
from welvet.cuda_b200 import decode as D

FAKE = 4096  # never dereferenced: every call below is refused first


def desc(**kw):
    base = dict(dtype=3, num_heads=8, num_kv_heads=2, head_dim=64, page_size=16, num_pages=10, num_seqs=2, pages_per_seq=4,
                k_pages=FAKE, v_pages=FAKE, k_strides=(ctypes.c_int64 * 3)(2048, 128, 64),
                v_strides=(ctypes.c_int64 * 3)(2048, 128, 64), k_scale=1.0, v_scale=1.0, page_table=FAKE, table_stride=4, lens=FAKE)
    base.update(kw)
    return D._KvDesc(**base)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=9), 2), (dict(dtype=0), 2), (dict(dtype=5), 2), (dict(num_heads=7), 1), (dict(num_heads=0), 1), (dict(num_kv_heads=0), 1),
    (dict(head_dim=0), 1), (dict(head_dim=257), 2), (dict(page_size=0), 1), (dict(num_pages=0), 1), (dict(num_seqs=0), 1),
    (dict(pages_per_seq=-1), 1), (dict(pages_per_seq=1 << 28), 2), (dict(num_seqs=70000), 2), (dict(table_stride=3), 1),
    (dict(page_table=None), 1), (dict(lens=None), 1), (dict(positions=FAKE), 1), (dict(k_scale=0.0), 1), (dict(v_scale=-1.0), 1),
    (dict(k_scale=float("inf")), 1), (dict(k_pages=None), 1), (dict(v_pages=None), 1), (dict(k_pages=FAKE + 1), 1),
    (dict(k_strides=(ctypes.c_int64 * 3)(2048, 32, 64)), 1), (dict(v_strides=(ctypes.c_int64 * 3)(2048, 128, -64)), 1),
    (dict(v_strides=(ctypes.c_int64 * 3)(0, 128, 64)), 1),
])
def test_cache_descriptions(kw, code):
    h = ctypes.c_void_p()
    st = W.lib().welvet_b200_kv_create(ctypes.byref(desc(**kw)), ctypes.byref(h))
    assert st.code == code and st.message.startswith(b"kv") and not h


def test_nil_handles():
    L = W.lib()
    assert L.welvet_b200_kv_create(None, None).code == 1
    assert L.welvet_b200_kv_append(None, 1, FAKE, 1, FAKE, 1, None, 0, None, 0, None, 0.0, None, None, None).code == 1
    assert L.welvet_b200_kv_attend(None, FAKE, 1, FAKE, 1, 0.0, 0, 0, 0, None, None).code == 1
    assert L.welvet_b200_kv_evict(None, 1, 1, 0, 0, None, None, None, None).code == 1
    assert L.welvet_b200_kv_check_error(None, None).code == 1
    assert L.welvet_b200_gdense_execute_device(None, 1, FAKE, 1, None, FAKE, None).code == 1
    assert L.welvet_b200_mha_decode_device(None, None, FAKE, None, FAKE, 0, None).code == 1
    assert L.welvet_b200_mha_prefill_device(None, None, 0, 1, FAKE, None, FAKE, None).code == 1
    L.welvet_b200_kv_release(None)
    L.welvet_b200_gdense_release(None)


@pytest.mark.parametrize("args,code", [
    ((0, 4, 64, 14, 2), 1), ((64, 0, 64, 14, 2), 1), ((64, 4, 48, 14, 2), 2), ((64, 4, 0, 14, 2), 2), ((64, 4, -64, 14, 2), 2),
    ((64, 4, 64, 9, 2), 2), ((64, 4, 64, 16, 1), 2),
])
def test_group_shapes(args, code):
    L = W.lib()
    st = L.welvet_b200_group_quantize(*args, FAKE, FAKE, FAKE, FAKE, None)
    assert st.code == code
    h = ctypes.c_void_p()
    st = L.welvet_b200_gdense_mount(*args, -1, FAKE, FAKE, FAKE if args[3] == 15 else None, 1, None, 0, ctypes.byref(h))
    assert st.code == code and not h


def test_group_arguments():
    L = W.lib()
    h = ctypes.c_void_p()
    m = lambda code, zeros, act=-1, bias=None, n=0: L.welvet_b200_gdense_mount(  # noqa: E731
        64, 4, 64, code, 2, act, FAKE, FAKE, zeros, 1, bias, n, ctypes.byref(h)).code
    assert m(15, None) == 1 and m(14, FAKE) == 1 and m(16, None, act=7) == 1 and m(16, None, n=3) == 1
    assert L.welvet_b200_group_quantize(64, 4, 64, 15, 2, FAKE, FAKE, FAKE, None, None).code == 1


def test_positions_need_a_seen_of_their_own():
    h = ctypes.c_void_p()
    st = W.lib().welvet_b200_kv_create(ctypes.byref(desc(positions=FAKE, seen=FAKE, lens=FAKE)), ctypes.byref(h))
    assert st.code == 1 and b"of its own" in st.message and not h


@pytest.mark.parametrize("in_,out", [((1 << 31) - 1, 16), (64, (1 << 31) - 1), ((1 << 30) + 1, 16)])
def test_group_sizes_past_the_index_range(in_, out):
    L = W.lib()
    assert L.welvet_b200_group_quantize(in_, out, 64, 14, 2, FAKE, FAKE, FAKE, None, None).code == 2
    h = ctypes.c_void_p()
    assert L.welvet_b200_gdense_mount(in_, out, 64, 14, 2, -1, FAKE, FAKE, None, 1, None, 0, ctypes.byref(h)).code == 2 and not h


def test_nil_handles_of_a_step_with_flags():
    assert W.lib().welvet_b200_mha_decode_active_device(None, None, FAKE, None, FAKE, 0, FAKE, None).code == 1


SHAPES = [(1, 1), (16, 64), (100, 130), (1024, 4096), (4096, 4096), (14336, 4096), (4096, 14336), (14331, 4090), (40, 16385), (256, 4609),
          (256, 17400), (38100, 600), (19024, 4609), (65536, 16384), (37888, 256), (3000, 100000), (500000, 64)]


@pytest.mark.parametrize("rows", range(1, 9))
@pytest.mark.parametrize("out,in_", SHAPES)
def test_group_plans(out, in_, rows):
    """What the kernel relies on: every slab has a chunk, every warp of a block a record, x and the sums
    that wait fit shared memory, runs that are whole row groups are no more than there are."""
    for code in (14, 15, 16):
        p = D.gdense_plan(in_, out, 64, code, rows)
        assert p["row_groups"] == -(-out // 16) and p["chunks"] == -(-in_ // 256)
        assert 0 < p["slabs"] * p["slab_chunks"] - p["chunks"] + 1 <= p["slab_chunks"]  # the last slab has a chunk
        assert p["slabs"] * p["slab_blocks"] <= 148 or p["slabs"] > 148
        last = p["chunks"] - (p["slabs"] - 1) * p["slab_chunks"]
        assert p["runs"] == p["slab_blocks"] * (16 if p["solo"] else 1)
        if p["whole"]:
            assert not p["solo"] and p["runs"] <= p["row_groups"] and p["cut"] == 0
        elif p["slab_blocks"] > 1:
            assert p["row_groups"] * last >= 16 * p["slab_blocks"]
        assert p["cut"] <= p["slabs"] * (p["runs"] - 1) and p["smem"] <= 227 * 1024
    for bad in (dict(rows=0), dict(rows=9), dict(sms=0), dict(group=48), dict(code=9), dict(out=0)):
        with pytest.raises(ValueError):
            D.gdense_plan(**{**dict(in_features=in_, out=out, group=64, code=14, rows=rows), **bad})
