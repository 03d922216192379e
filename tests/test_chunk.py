"""The operators of prompts in chunks without a GPU: rotary frequencies, the
refusals that need no device, the definitions of tests/chunk_case.py on inputs
small enough to follow by hand."""
import ctypes as C

import numpy as np
import pytest
import torch

from styx_b200 import StyxError, _lib, ops
from tests.chunk_case import Tables, chunk_ref, freqs_ref, turned_ref


@pytest.fixture(scope="module", autouse=True)
def built():
    from styx_b200 import build
    build.build()


@pytest.mark.parametrize("n,base,kw", [
    (128, 1e6, {}), (64, 1e4, {}), (2, 1e4, {}), (80, 5e5, dict(scaling="linear", factor=8.0)),
    (128, 1e6, dict(scaling="yarn", factor=4.0, orig=32768)), (64, 1e4, dict(scaling="yarn", factor=16.0, orig=4096)),
    (96, 1e4, dict(scaling="yarn", factor=1.0, orig=2048)),
    (128, 5e5, dict(scaling="yarn", factor=2.0, orig=8, fast=3.0, slow=2.9)),       # all pairs slow: lo = hi = 0
    (64, 1e4, dict(scaling="yarn", factor=4.0, orig=4096, fast=1.0, slow=32.0)),     # the edges the other way round
])
@pytest.mark.parametrize("with_factors", [False, True])
def test_frequencies(n, base, kw, with_factors):
    factors = np.linspace(1, 8, n // 2).astype(np.float32) if with_factors else None
    exp, grow = freqs_ref(n, base, factors=factors, **kw)
    named = {"orig": "orig_ctx", "fast": "beta_fast", "slow": "beta_slow"}
    got, g = ops.Rope.frequencies(n, base, factors=None if factors is None else torch.from_numpy(factors),
                                  **{named.get(k, k): v for k, v in kw.items()})
    # a power, a logarithm or two, a few products in 64 bits
    assert np.max(np.abs(got.numpy() / exp - 1)) < 1e-13 and abs(g - grow) <= 2 ** -24 * grow


@pytest.mark.parametrize("kw", [dict(n_dims=0), dict(n_dims=63), dict(n_dims=-2), dict(n_dims=5000), dict(base=1.0),
                                dict(base=float("nan")), dict(base=float("inf")),
                                dict(scaling="linear", factor=0.5), dict(scaling="linear", factor=float("nan")),
                                dict(scaling="yarn", factor=4.0), dict(scaling="yarn", factor=4.0, orig_ctx=-1),
                                dict(scaling="yarn", factor=4.0, orig_ctx=100, beta_fast=0.0),
                                dict(factors=torch.zeros(32)), dict(factors=torch.full((32,), float("inf")))])
def test_frequencies_refused(kw):
    with pytest.raises(StyxError):
        ops.Rope.frequencies(**{"n_dims": 64, "base": 1e4, **kw})


def test_frequency_arguments_refused():
    with pytest.raises(ValueError, match="scaling"):
        ops.Rope.frequencies(64, 1e4, "ntk")
    with pytest.raises(ValueError, match="factors"):
        ops.Rope.frequencies(64, 1e4, factors=torch.ones(64))
    L, g = _lib.lib(), C.c_float()
    assert L.styx_rope_freqs(None, None, None, C.byref(g)) == _lib.STYX_EINVAL
    assert L.styx_rope_freqs(C.byref(_lib.RopeParams(64, 3, 1e4, 1, 1, 1, 1)), None, torch.zeros(32, dtype=torch.float64).data_ptr(),
                             C.byref(g)) == _lib.STYX_EINVAL


def test_null_contexts_refused():
    L, n = _lib.lib(), C.c_uint64()
    assert L.styx_paged_plan(*[None] * 4, 1, *[None] * 9) == _lib.STYX_EINVAL
    assert L.styx_paged_chunk_workspace_bytes(None, None, 8, 0, C.byref(n)) == _lib.STYX_EINVAL
    assert L.styx_paged_attend_chunk(None, None, None, 1, 1, 0, None, 0, None, 1.0, 0, None, None, None, 0) == _lib.STYX_EINVAL
    assert L.styx_paged_append_rope(None, None, None, 1, 1, None, 0, None, 0, None, 0, None, None, 0.0, None, None, None,
                                    None, 0, None) == _lib.STYX_EINVAL


def test_cpu_tensors_refused():
    i = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.PagedPlan(torch.zeros(4, 4, dtype=torch.int32), 16, i, 8)


def test_chunk_definition():
    k, v = np.zeros((3, 1, 2)), np.arange(6.0).reshape(3, 1, 2)
    out, lse, mag = chunk_ref(np.ones((2, 1, 2)), [0, 2], [k], [v], 1.0)
    assert np.allclose(out[:, 0], [[1, 2], [2, 3]]) and np.allclose(lse[:, 0], np.log([2, 3])) and np.allclose(mag, out)
    out, _, _ = chunk_ref(np.ones((2, 1, 2)), [0, 2], [k], [v], 1.0, window=1)
    assert np.allclose(out[:, 0], [[2, 3], [4, 5]])


def test_turn_definition():
    x = np.array([[[1.0, 0, 0, 0, 5, 6]]])
    f = np.array([1.0, 0.5])
    assert np.allclose(turned_ref(x, None, np.array([2]), f, 4, False, 3.0, 0), [[[3 * np.cos(2), 0, 3 * np.sin(2), 0, 5, 6]]])
    assert np.allclose(turned_ref(x, None, np.array([2]), f, 4, True, 1.0, 0), [[[np.cos(2), np.sin(2), 0, 0, 5, 6]]])


def test_plan_definition():
    t = Tables(np.random.default_rng(0), 3, 4, 2, 6, [3, 0, 1], [2, 1, 1])
    ids = t.table.copy()
    stack = t.free[:t.n_free].tolist()
    # the second is done: its page is the first to be taken; the third finds two of its three pages
    start, seq, row, pos = t.plan([2, 0, 5], 8)
    assert start.tolist() == [0, 2, 2, 7] and row.tolist() == [3, 4, 1, 2, 3, 4, 5, -1]
    assert t.table[0, 2] == ids[1, 0] and t.table[2, 1:3].tolist() == stack[::-1] and t.n_free == 0
    assert t.lens == [5, 0, 6] and t.held == [3, 0, 3] and pos.tolist()[:3] == [3, 4, 15] and seq.tolist() == [0, 0, 2, 2, 2, 2, 2, 0]


def test_batch_decoder_refuses_chunks_it_cannot_have():
    from styx_b200.decode import DecodeParams
    from styx_b200.serve import BatchDecoder
    hp = DecodeParams(1, 512, 8, 2, 64, 256, 16, 4, 1024)
    with pytest.raises(ValueError, match="chunks"):
        BatchDecoder(hp, None, [], None, None, 4, 64, chunk=-1)
    with pytest.raises(ValueError, match="budget"):
        BatchDecoder(hp, None, [], None, None, 4, 64, chunk=8, budget=32, n_recent=8, n_sink=4)
