"""The host side of include/styx_serve.h without a GPU: workspace sizes and
the refusals that need no device; the 64-bit definitions of
tests/paged_case.py on inputs small enough to follow by hand."""
import ctypes as C

import numpy as np
import pytest
import torch

from styx_b200 import _lib, ops
from tests.paged_case import attend_ref, evict_ref, rope_norm_ref


def kv(**over):
    a = dict(k=0, v=0, page_stride=2 * 16 * 64, table=0, lens=0, dtype=_lib.F16, n_pages=10, page_size=16, n_kv_heads=2,
             head_dim=64, n_seqs=3, max_pages=4, table_stride=4)
    a.update(over)
    return _lib.PagedKv(*a.values())


@pytest.fixture(scope="module", autouse=True)
def built():
    from styx_b200 import build
    build.build()


def test_evict_workspace_bytes():
    n = C.c_uint64()
    assert _lib.lib().styx_paged_evict_workspace_bytes(C.byref(kv()), 100, C.byref(n)) == 0
    assert n.value >= 2 * 3 * 2 * 100 * 4


@pytest.mark.parametrize("over", [dict(dtype=8), dict(head_dim=60), dict(head_dim=0), dict(head_dim=512),
                                  dict(dtype=_lib.F32, head_dim=6), dict(page_size=0), dict(page_size=24),
                                  dict(page_size=8192), dict(n_kv_heads=0), dict(n_seqs=0), dict(n_seqs=70000),
                                  dict(n_pages=0), dict(max_pages=0), dict(table_stride=3), dict(page_stride=2047),
                                  dict(page_stride=2049), dict(max_pages=1 << 28, table_stride=1 << 28)])
def test_cache_descriptions_refused(over):
    n = C.c_uint64()
    assert _lib.lib().styx_paged_evict_workspace_bytes(C.byref(kv(**over)), 100, C.byref(n)) == _lib.STYX_EINVAL
    assert _lib.lib().styx_last_error()


def test_null_arguments_refused():
    L, n = _lib.lib(), C.c_uint64()
    assert L.styx_paged_evict_workspace_bytes(None, 1, C.byref(n)) == _lib.STYX_EINVAL
    assert L.styx_paged_evict_workspace_bytes(C.byref(kv()), 0, C.byref(n)) == _lib.STYX_EINVAL
    assert L.styx_sample(None, None, None, 1, 1, 1, None, None, None, None, None, None, None) == _lib.STYX_EINVAL
    assert L.styx_paged_attend_workspace_bytes(None, C.byref(kv()), 8, 0, C.byref(n)) == _lib.STYX_EINVAL


def test_cpu_tensors_refused():
    x = torch.zeros(2, 8)
    with pytest.raises(ValueError):
        ops.sample(x, torch.zeros(2))
    p = torch.zeros(4, 2, 16, 64)
    with pytest.raises(ValueError):
        ops.PagedKV(p, p, torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))


def test_evict_definition():
    acc = np.array([5, 1, 1, 9, 2, 1, 7, 3], np.float32)
    pos = np.arange(8, dtype=np.int32)
    # three stay: row 7 (newest), rows 3 and 6 by weight; 6 and 7 fill the places 0 and 1, 3 fills 2
    assert evict_ref(acc, pos, 8, 8, 3, 1, 0).tolist() == [3, 6, 7]
    assert evict_ref(acc, pos, 8, 8, 4, 0, 1).tolist() == [0, 6, 7, 3]
    assert evict_ref(acc, pos, 3, 8, 4, 0, 1).tolist() == [0, 1, 2]
    assert evict_ref(np.zeros(5, np.float32), pos, 5, 8, 2, 0, 0).tolist() == [0, 1]


def test_attend_definition():
    k, v = np.zeros((3, 1, 2)), np.arange(6.0).reshape(3, 1, 2)
    out, lse, w = attend_ref(np.ones((1, 2, 2)), [k], [v], 1.0)
    assert np.allclose(out[0, 0], [2, 3]) and np.allclose(lse, np.log(3)) and np.allclose(w[0], 2 / 3)
    out, _, w = attend_ref(np.ones((1, 2, 2)), [k], [v], 1.0, window=1)
    assert np.allclose(out[0, 0], [4, 5]) and np.allclose(w[0], [[0, 0, 2]])


def test_rope_definition():
    x = np.array([[[1.0, 0, 0, 0]]])
    y = rope_norm_ref(x, None, np.array([2]), 100.0, 0)
    assert np.allclose(y, [[[np.cos(2), 0, np.sin(2), 0]]])


def test_batch_decoder_refuses_what_it_cannot_hold():
    from styx_b200.decode import DecodeParams
    from styx_b200.serve import BatchDecoder
    hp = DecodeParams(1, 512, 8, 2, 64, 256, 16, 4, 1024)
    with pytest.raises(ValueError, match="sequences"):
        BatchDecoder(hp, None, [], None, None, 0, 64)
    with pytest.raises(ValueError, match="sequences"):
        BatchDecoder(hp, None, [], None, None, 65, 64)
    with pytest.raises(ValueError, match="budget"):
        BatchDecoder(hp, None, [], None, None, 4, 64, budget=16, n_recent=14, n_sink=4)


def test_caches_of_different_devices_do_not_share_workspaces():
    a, b = (ops.PagedKV.__new__(ops.PagedKV) for _ in range(2))
    for index, o in enumerate((a, b)):
        o.k, o.table = torch.zeros(4, 2, 16, 64), torch.zeros(1, 4, dtype=torch.int32)
        o.index, o._attend_ws, o._evict_ws = index, {}, []
    with pytest.raises(ValueError, match="share_workspaces"):
        a.share_workspaces(b)
    b.index = 0
    a.share_workspaces(b)
    assert a._attend_ws is b._attend_ws and a._evict_ws is b._evict_ws


def test_evict_workspace_goes_by_the_rows_there_are():
    """A budget beyond a sequence's rows moves nothing: from whole slices of 4096 rows on it takes no more room."""
    L, n, most = _lib.lib(), C.c_uint64(), C.c_uint64()
    for pages, slices in ((4, 1), (256, 1), (257, 2)):     # 64, 4096 and 4112 rows
        of = kv(max_pages=pages, table_stride=pages)
        assert L.styx_paged_evict_workspace_bytes(C.byref(of), 4096 * slices, C.byref(most)) == 0
        for budget in (4096 * slices + 1, 10 ** 9, 2 ** 31 - 1):
            assert L.styx_paged_evict_workspace_bytes(C.byref(of), budget, C.byref(n)) == 0
            assert n.value == most.value < 2 * 6 * 4096 * slices * 4 + 1024
        assert L.styx_paged_evict_workspace_bytes(C.byref(of), 63, C.byref(n)) == 0 and n.value < most.value
