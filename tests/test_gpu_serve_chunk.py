"""styx_b200.serve with prompts in chunks (plan, append, attend_chunk as one
path) against the oracle and against prompts a token at a time."""
import numpy as np
import pytest
import torch

from styx_b200 import ops, serve
from tests.decode_case import make_model, oracle_greedy, write_gguf
from tests.test_gpu_decode import gpu_model

pytestmark = pytest.mark.gpu

PROMPTS = [[5, 17, 99], [640], [3, 1, 4, 1, 5, 9, 2, 6, 5, 3, 5, 8, 9], [1000, 2, 77]]


def decoder(m, **kw):
    return serve.BatchDecoder.of(gpu_model(m, 8), len(PROMPTS), kw.pop("n_ctx", 64), **kw)


@pytest.mark.parametrize("hd,page,chunk", [(64, 16, 1), (64, 16, 5), (128, 4, 7), (128, 16, 512)])
def test_greedy_tokens_are_those_of_the_oracle(hd, page, chunk):
    m = make_model(0, hd=hd)
    expect = [oracle_greedy(m, p, 12) for p in PROMPTS]
    d = decoder(m, page=page, cache=torch.float32, moe_batch=False, chunk=chunk)
    assert d.generate(PROMPTS, 12) == expect
    assert d.generate(PROMPTS, 12) == expect                     # from the start again
    # pages and lengths as the host and the device know them
    assert d.lens.tolist() == d.rows == d.pos.tolist()
    used = [p for ps in d.pages for p in ps]
    assert sorted(used + d.free) == list(range(d.n_pages)) and [len(ps) for ps in d.pages] == [-(-n // page) for n in d.rows]
    assert [d.table[b, :len(ps)].tolist() for b, ps in enumerate(d.pages)] == d.pages


@pytest.mark.parametrize("cache", ["f16", "bf16"])
def test_logits_of_16_bit_rows_and_batched_experts(cache):
    """The bound of the step a token at a time: rows to 2^-11 (2^-8) and
    experts to 1e-3 of themselves, two layers, each update no larger than the
    residual stream."""
    m = make_model(1)
    one = gpu_model(m, 64)
    d = decoder(m, cache=serve.CACHE_TYPES[cache], chunk=6)
    assert d.moe_batch
    tol = 4 * ((2.0 ** -11 if cache == "f16" else 2.0 ** -8) + 1e-3)
    got = d.prefill(PROMPTS).clone()
    more = d.prefill([[7, 8], [], [9], []]).clone()               # and on from there
    for b, (p, add) in enumerate(zip(PROMPTS, ([7, 8], [], [9], []))):
        one.reset()
        for t in p:
            ref = one.forward_token(t)
        assert (got[b] - ref).abs().max() <= tol * ref.abs().max()
        if add:
            for t in add:
                ref = one.forward_token(t)
            assert (more[b] - ref).abs().max() <= tol * ref.abs().max()
    assert d.rows == [5, 1, 14, 3] == d.lens.tolist()
    d.kv[0].ctx.check_device_error()


def test_rotary_forms():
    """The model's own base said as a Rope changes nothing but roundings; a
    scaled one changes what later positions see; chunks and steps agree."""
    m = make_model(0, hd=64)
    hp = gpu_model(m, 8).hp
    kw = dict(cache=torch.float32, moe_batch=False)
    plain = decoder(m, chunk=9, **kw).prefill(PROMPTS).clone()
    same = decoder(m, chunk=9, rope=ops.Rope(64, hp.rope_base), **kw).prefill(PROMPTS).clone()
    assert (plain - same).abs().max() <= 1e-4 * plain.abs().max()
    rope = ops.Rope(64, hp.rope_base, scaling="yarn", factor=4.0, orig_ctx=8)
    scaled = decoder(m, chunk=9, rope=rope, **kw)
    a = scaled.prefill(PROMPTS).clone()
    assert (a - plain).abs().max() > 1e-2 * plain.abs().max()
    steps = decoder(m, rope=rope, **kw)
    for b, p in enumerate(PROMPTS):
        steps.reset()
        for t in p:
            steps.tok.fill_(t)
            got = steps.step(1)[0].clone()
        assert (got - a[b]).abs().max() <= 1e-4 * a[b].abs().max()


def test_what_does_not_fit_is_refused_and_changes_nothing():
    m = make_model(0, n_layers=1)
    d = decoder(m, n_ctx=12, page=4, chunk=8)
    with pytest.raises(ValueError, match="cache full"):
        d.prefill(PROMPTS)
    d = decoder(m, page=4, n_pages=5, chunk=8)
    with pytest.raises(ValueError, match="no page left"):
        d.prefill(PROMPTS)
    with pytest.raises(ValueError, match="prompts"):
        d.prefill(PROMPTS[:2])
    assert d.rows == [0] * 4 and len(d.free) == 5 and not d.lens.any()
    d.prefill([[1], [2], [3, 4, 5, 6, 7], []])
    assert d.rows == [1, 1, 5, 0] and len(d.free) == 1
    with pytest.raises(ValueError, match="chunk"):
        decoder(m).prefill(PROMPTS)


def test_command_line(tmp_path, capsys):
    m = make_model(0)
    path = str(tmp_path / "m.gguf")
    write_gguf(m, path)
    argv = [path, "-n", "12", "--ctx", "64", "--cache", "f32", "--experts", "f32", "--chunk", "6"]
    for p in PROMPTS:
        argv += ["--prompt", ",".join(map(str, p))]
    assert serve.main(argv) == 0
    out = [[int(t) for t in o.split(",")] for o in capsys.readouterr().out.split()]
    assert out == [oracle_greedy(m, p, 12) for p in PROMPTS]
    assert serve.main(argv + ["--rope-scaling", "yarn", "--rope-factor", "4", "--rope-orig-ctx", "16"]) == 0
    assert len(capsys.readouterr().out.split()) == 4
