"""styx_b200.serve (append, attend, evict and sample as one batched decode
step) against the oracle and the single-sequence decode step over the same
weights."""
import numpy as np
import pytest
import torch

from styx_b200 import serve
from tests.decode_case import make_model, oracle_greedy, write_gguf
from tests.test_gpu_decode import gpu_model

pytestmark = pytest.mark.gpu

PROMPTS = [[5, 17, 99], [640], [3, 1, 4, 1, 5, 9, 2], [1000, 2, 77]]


def decoder(m, **kw):
    return serve.BatchDecoder.of(gpu_model(m, 8), len(PROMPTS), kw.pop("n_ctx", 64), **kw)


@pytest.mark.parametrize("hd,page", [(64, 16), (128, 4)])
def test_greedy_tokens_are_those_of_the_oracle(hd, page):
    m = make_model(0, hd=hd)
    expect = [oracle_greedy(m, p, 12) for p in PROMPTS]
    # f32 rows and f32 experts: the same arithmetic up to the order of sums
    d = decoder(m, page=page, cache=torch.float32, moe_batch=False)
    assert d.generate(PROMPTS, 12) == expect
    assert d.generate(PROMPTS, 12) == expect                     # from the start again
    # a budget that nothing reaches changes nothing
    d = decoder(m, page=page, cache=torch.float32, moe_batch=False, budget=32, n_recent=8, n_sink=2)
    assert d.generate(PROMPTS, 12) == expect


@pytest.mark.parametrize("cache", ["f16", "bf16"])
def test_logits_of_16_bit_rows_and_batched_experts(cache):
    """K and V rounded to 2^-11 (bf16: 2^-8) of themselves and the experts'
    operands to f16 (1e-3 of a block's largest update): two layers, each update
    no larger than the residual stream, stay within 4 (2^-11 + 1e-3) and
    4 (2^-8 + 1e-3) of the largest logit."""
    m = make_model(1)
    one = gpu_model(m, 64)
    d = decoder(m, cache=serve.CACHE_TYPES[cache])
    assert d.moe_batch
    tol = 4 * ((2.0 ** -11 if cache == "f16" else 2.0 ** -8) + 1e-3)
    rng = np.random.default_rng(2)
    toks = rng.integers(0, m.hp["n_vocab"], (9, len(PROMPTS)))
    got = []
    for t in toks:
        d.tok.copy_(torch.from_numpy(t.astype(np.int32)))
        got.append(d.step().cpu().numpy().copy())
    for b in range(len(PROMPTS)):
        one.reset()
        for i, t in enumerate(toks):
            ref = one.forward_token(int(t[b])).cpu().numpy()
            assert np.abs(got[i][b] - ref).max() <= tol * np.abs(ref).max()


def test_a_budget_bounds_rows_and_pages():
    m = make_model(2)
    budget, recent, sinks, page = 24, 8, 2, 8
    d = decoder(m, page=page, cache=torch.float16, budget=budget, n_recent=recent, n_sink=sinks, n_pages=4 * 4)
    out = d.generate(PROMPTS, 60, temperature=0.8, top_k=50, top_p=0.95, min_p=0.01, seed=3)
    assert all(len(o) == 60 and all(0 <= t < m.hp["n_vocab"] for t in o) for o in out)
    lens = d.lens.tolist()
    assert lens == d.rows and all(budget <= n < budget + page for n in lens)
    used = [p for ps in d.pages for p in ps]
    assert sorted(used + d.free) == list(range(16)) and [len(ps) for ps in d.pages] == [-(-n // page) for n in lens]
    assert [d.table[b, :len(ps)].tolist() for b, ps in enumerate(d.pages)] == d.pages
    for b, p in enumerate(sorted(PROMPTS, key=lambda p: -len(p))):
        nxt = len(p) + 59
        assert d.pos[b].item() == nxt
        for li in range(m.hp["n_layers"]):
            rows = d.row_pos[li][b, :, :lens[b]].cpu().numpy()
            for r in rows:      # no position twice; the first ones and the last ones are there
                assert len(set(r.tolist())) == len(r)
                assert set(range(sinks)) | set(range(nxt - recent, nxt)) <= set(r.tolist())
    # the same settings and seed draw the same tokens; another seed others
    assert d.generate(PROMPTS, 60, temperature=0.8, top_k=50, top_p=0.95, min_p=0.01, seed=3) == out
    assert d.generate(PROMPTS, 60, temperature=0.8, top_k=50, top_p=0.95, min_p=0.01, seed=4) != out


def test_full_caches_and_pools_are_refused():
    m = make_model(0, n_layers=1)
    d = decoder(m, n_ctx=8, page=4)
    with pytest.raises(ValueError, match="cache full"):
        d.generate(PROMPTS, 4)
    d = decoder(m, page=4, n_pages=5)
    with pytest.raises(ValueError, match="no page left"):
        d.generate(PROMPTS, 20)
    with pytest.raises(ValueError, match="prompts"):
        d.generate(PROMPTS[:2], 4)


def test_command_line(tmp_path, capsys):
    m = make_model(0)
    path = str(tmp_path / "m.gguf")
    write_gguf(m, path)
    argv = [path, "-n", "10", "--ctx", "64", "--cache", "f32"]
    for p in PROMPTS[:2]:
        argv += ["--prompt", ",".join(map(str, p))]
    assert serve.main(argv) == 0
    out = capsys.readouterr().out.split()
    assert len(out) == 2 and all(len(o.split(",")) == 10 for o in out)


def test_a_step_of_some_sequences_leaves_the_others_as_they_are():
    m = make_model(2)
    d = decoder(m, page=8, cache=torch.float16, budget=24, n_recent=8, n_sink=2)
    whole = decoder(m, page=8, cache=torch.float16, budget=24, n_recent=8, n_sink=2)
    rng = np.random.default_rng(4)
    toks = [torch.from_numpy(rng.integers(0, m.hp["n_vocab"], 4).astype(np.int32)) for _ in range(5)]

    def step(dec, t, n=None):
        dec.tok.copy_(t)
        return dec.step(n).clone()

    for t in toks[:3]:
        step(d, t)
        step(whole, t)
    L = m.hp["n_layers"]
    acc, pos, rows = [a.clone() for a in d.acc[:L]], [p.clone() for p in d.row_pos[:L]], list(d.rows)
    used = torch.tensor([p for ps in d.pages[2:] for p in ps], device=d.device)
    pool = d.pool[:, :, used].clone()
    got = step(d, toks[3], 2)
    # (other sums than a step of all four: the bound of the 16-bit rows and experts above)
    ref = step(whole, toks[3])[:2]
    assert (got - ref).abs().max() <= 4 * (2.0 ** -11 + 1e-3) * ref.abs().max()
    for li in range(L):
        assert torch.equal(d.acc[li][2:], acc[li][2:]) and not torch.equal(d.acc[li][:2], acc[li][:2])
        assert torch.equal(d.row_pos[li][2:], pos[li][2:])
    assert torch.equal(d.pool[:, :, used].view(torch.int16), pool.view(torch.int16))
    assert d.rows == [rows[0] + 1, rows[1] + 1] + rows[2:] == d.lens.tolist() and d.pos.tolist() == d.rows
    # evicting with sequences that the last step left out reaches them too
    d.budget = 3
    d.n_recent, d.n_sink = 1, 1
    d.evict()
    assert d.lens.tolist() == [3] * 4 == d.rows
    # a step of all of them goes on from there
    assert step(d, toks[4]).isfinite().all() and d.lens.tolist() == [4] * 4
    d.kv[0].ctx.check_device_error()


@pytest.mark.parametrize("kind", ["pages", "rows"])
def test_a_refused_step_changes_nothing(kind):
    """The third of four sequences needs the page (row) that is not there: the first two have taken none either, and
    the step goes through once there is room."""
    m = make_model(0, n_layers=1)
    d = decoder(m, n_ctx=8, page=4, n_pages=6 if kind == "pages" else None)
    for i in range(4):
        d.step()                                           # four rows each: one full page
    if kind == "rows":
        d.lens[2], d.rows[2] = 8, 8                        # the third is full
        d.pages[2].append(d.free.pop())
    before = (list(d.rows), [list(p) for p in d.pages], list(d.free), d.lens.tolist(), d.table.tolist(), d.pos.tolist())
    for _ in range(3):
        with pytest.raises(ValueError, match="sequence 2: no page left" if kind == "pages" else "sequence 2: KV cache full"):
            d.step()
        assert before == (list(d.rows), [list(p) for p in d.pages], list(d.free), d.lens.tolist(), d.table.tolist(),
                          d.pos.tolist())
    for n in (0, -1, 5):
        with pytest.raises(ValueError, match="sequences"):
            d.step(n)
    d.step(2)
    assert d.lens.tolist() == d.rows and d.rows[:2] == [5, 5]
    d.kv[0].ctx.check_device_error()


def test_command_line_in_f32_gives_the_oracles_tokens(tmp_path, capsys):
    m = make_model(0)
    path = str(tmp_path / "m.gguf")
    write_gguf(m, path)
    argv = [path, "-n", "12", "--ctx", "64", "--cache", "f32", "--experts", "f32"]
    for p in PROMPTS:
        argv += ["--prompt", ",".join(map(str, p))]
    assert serve.main(argv) == 0
    out = [[int(t) for t in o.split(",")] for o in capsys.readouterr().out.split()]
    assert out == [oracle_greedy(m, p, 12) for p in PROMPTS]
